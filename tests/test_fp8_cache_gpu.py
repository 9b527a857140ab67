"""The 8-bit cache on the device, against its definition in 64 bits (plain_fp8_cache)."""
import math

import pytest
import torch

import plain_fp8_cache as plain
import test_fp8_cache as host
from ferrox_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


CHOICE = ops.fp8_token_by_token


@pytest.fixture(autouse=True)
def tiled(monkeypatch):
    """Steps this small would go through the decode kernel; the tests are of the others (test_prompts_as_chosen: as they come)."""
    monkeypatch.setattr(ops, "fp8_token_by_token", lambda kind, entries, *a: all(n <= ops.FP8_FEW_TOKENS for n, _ in entries))


class Cache:
    """A cache of ``lens`` positions for each request in scattered pages of a pool, and what it holds by the definition."""

    def __init__(self, lens, G, D, P, seed, extra_pages=3, spread=0.0, pool=None, slots=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.G, self.D, self.P = lens, G, D, P
        need = [-(-n // P) for n in lens]
        n_pages = pool or sum(need) + extra_pages
        order = torch.randperm(n_pages, generator=g)
        if pool:
            order = torch.arange(n_pages - 1, -1, -1)                       # (a large pool: its last pages)
        self.slots = torch.randperm(len(lens) + 2, generator=g)[:len(lens)].to(torch.int32)
        self.table = torch.full((len(lens) + 2, max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[self.slots[b], :n] = order[at:at + n].to(torch.int32)
            at += n
        self.used = order[:at]

        def rows():
            x = torch.randn(at, G, P, D, generator=g, dtype=torch.float64)
            if spread:
                x = x * torch.exp2(torch.round(spread * torch.randn(at, G, P, 1, generator=g, dtype=torch.float64)))
            return plain.quantise(x)

        (kv, ke), (vv, ve) = rows(), rows()
        self.dev = []
        for vals, exps in ((kv, ke), (vv, ve)):
            pages = torch.zeros(n_pages, G, P, D, dtype=torch.uint8, device=DEV)
            pages[self.used.to(DEV)] = vals.float().to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
            e = torch.zeros(n_pages, G, P, dtype=torch.uint8, device=DEV)
            e[self.used.to(DEV)] = exps.to(torch.uint8).to(DEV)
            self.dev.append((pages.view(torch.float8_e4m3fn), e))
        self.plain = (kv, ke, vv, ve)

    @property
    def operands(self):
        (k, ke), (v, ve) = self.dev
        return k, v, ke, ve, self.table.to(DEV), self.P

    def of(self, b, upto, which):
        """[positions, kv heads, dim] of request b and whether each has a page."""
        pages, e = self.dev[which]
        row = self.table[self.slots[b]]
        ids = row.long().clamp_min(0)
        return plain.held(pages.view(torch.uint8)[ids.to(DEV)].cpu(), e[ids.to(DEV)].cpu(),
                          torch.where(row >= 0, torch.arange(row.numel()), -1), upto)


def step(entries, slots):
    pos = torch.cat([torch.arange(s, s + n) for n, s in entries]).to(torch.int32).to(DEV)
    seq = torch.cat([torch.full((n,), b) for b, (n, _) in enumerate(entries)]).to(torch.int32).to(DEV)
    return pos, seq, slots.to(DEV)


def check(out, c, entries, q, H, window, scale, softcap, weight_error):
    """Every token's result against the definition.  A result is rounded once to its type (half a step); a weight is off by
    ``weight_error`` (what its kernel rounds it to) and by the errors of 32-bit scores: a dot product of D products and its
    scale (D + 8 roundings of at most half a step of the sum of their magnitudes), the cap (its own rounding and slope at most
    1), exp (its own 2 steps and the argument's 32-bit rounding, scores here being below 64 in size: 2^-18); n weights are added
    up in 32 bits above and below the fraction (n half steps each, at most 2^-24 * (n + 64))."""
    at = 0
    eps = torch.finfo(out.dtype).eps / 2
    for b, (n, start) in enumerate(entries):
        if n == 0:
            continue
        k, there = c.of(b, start + n, 0)
        v, _ = c.of(b, start + n, 1)
        want, mag, most = plain.attention(q[at:at + n, :H * c.D].double().cpu().reshape(n, H, c.D), k, v, there, range(start, start + n), H,
                                          window, scale, softcap)
        score = most * (c.D + 8) * 2.0 ** -24 + (2.0 ** -22 * softcap if softcap else 0.0)
        tol = eps * want.abs() + mag * (weight_error + 2 * score + 2.0 ** -18 + 2.0 ** -23 * (start + n + 64)) + 1e-37
        got = out[at:at + n].double().cpu().reshape(n, H, c.D)
        assert torch.equal(torch.isnan(got), torch.isnan(want)), f"request {b}: other elements are no numbers"
        off = torch.nan_to_num((got - want).abs() - tol, nan=-1.0)
        assert off.max() <= 0, f"request {b}: off by {float(torch.nan_to_num((got - want).abs()).max()):.3g}, {float(off.max()):.3g} too much"
        at += n


def rows(T, H, G, D, dtype, seed, extra=0, q_scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, (H + 2 * G) * D + extra, generator=g)
    x[:, :H * D] *= q_scale
    return x.to(dtype).to(DEV)


# ---- write and read -------------------------------------------------------------------------------------------------
def turned(x, pos, inv_freq, rot, pairing):
    """Heads [tokens, heads, D] rotated in 64 bits by 32-bit angles, as the definition of the rotary kernel says."""
    y = x.double().clone()
    ang = (pos.float()[:, None] * inv_freq[None]).double()
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    half = rot // 2
    ia, ib = (slice(0, rot, 2), slice(1, rot, 2)) if pairing else (slice(0, half), slice(half, rot))
    a, b = x.double()[..., ia], x.double()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P,extra", [(4, 2, 128, 16, 0), (2, 2, 64, 64, 8), (3, 1, 256, 32, 0), (6, 3, 48, 5, 0), (1, 1, 7, 3, 1), (2, 1, 128, 16, 3),
                                           (2, 2, 200, 7, 0), (28, 4, 128, 64, 0)])
def test_write_and_read_back_bit_for_bit(dtype, H, G, D, P, extra):
    lens = [1, 2 * P, 3 * P - 1]
    c = Cache(lens, G, D, P, 1)
    entries = [(1, 0), (P + 1, P - 1), (2, 3 * P - 3)]
    pos, seq, slots = step(entries, c.slots)
    T = pos.numel()
    qkv = rows(T, H, G, D, DTYPES[dtype], 2, extra)
    qkv[:, H * D:(H + 2 * G) * D] *= torch.exp2(torch.randint(-40, 40, (T, 1), generator=torch.Generator().manual_seed(3)).float()).to(DEV).to(qkv.dtype)
    before, pages = qkv.clone(), [(p.view(torch.uint8).clone(), e.clone()) for p, e in c.dev]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_kv_write_fp8(qkv, pos, seq, slots, None, 0, *c.operands, H, G, D, status=status)
    assert int(status) == 0 and torch.equal(qkv, before)
    k_out, v_out = (torch.full((T, G, D), 7.0, dtype=qkv.dtype, device=DEV) for _ in range(2))
    ops.read_kv_fp8(*c.operands, pos, seq, slots, k_out, v_out)
    for which, got in ((0, k_out), (1, v_out)):
        x = before[:, (H + which * G) * D:(H + which * G + G) * D].reshape(T, G, D).cpu()
        vals, exps = plain.quantise(x)
        assert torch.equal(got.double().cpu(), plain.values(vals, exps))
        # the bytes themselves lie in their places, and nothing else has changed
        page = c.table[c.slots[seq.cpu().long()].long(), pos.cpu().long() // P].long().to(DEV)
        p, e = pages[which]
        p[page, :, pos.long() % P] = vals.float().to(torch.float8_e4m3fn).view(torch.uint8).to(DEV)
        e[page, :, pos.long() % P] = exps.to(torch.uint8).to(DEV)
        now = c.dev[which]
        zero = (now[0].view(torch.uint8) & 127) == 0                        # (0 and -0 stand for the same)
        assert torch.equal(torch.where(zero, 0, now[0].view(torch.uint8)), torch.where((p & 127) == 0, 0, p)) and torch.equal(now[1], e)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,rot,pairing", [(128, 128, 0), (64, 64, 0), (256, 256, 0), (128, 64, 0), (64, 64, 1), (48, 32, 1), (96, 96, 0), (10, 6, 1)])
@pytest.mark.parametrize("table", [False, True])
def test_rotation_before_the_write(dtype, D, rot, pairing, table):
    H, G, P = 3, 2, 16
    c = Cache([40, 9], G, D, P, 4)
    pos, seq, slots = step([(17, 20), (3, 6)], c.slots)
    T = pos.numel()
    qkv = rows(T, H, G, D, DTYPES[dtype], 5)
    inv_freq = 10000.0 ** (-torch.arange(rot // 2).float() / (rot // 2))
    cos_sin = torch.empty(T, rot // 2, 2, device=DEV)
    ops.rope_table(pos, inv_freq.to(DEV), cos_sin)
    before = qkv.cpu()
    ops.rope_kv_write_fp8(qkv, pos, seq, slots, inv_freq.to(DEV), rot, *c.operands, H, G, D, cos_sin=cos_sin if table else None, pairing=pairing)
    heads = qkv.cpu().reshape(T, H + 2 * G, D)
    want = turned(before.reshape(T, -1, D)[:, :H + G], pos.cpu(), inv_freq, rot, pairing)
    mag = before.reshape(T, -1, D)[:, :H + G].double().abs().amax(-1, keepdim=True)
    # a rounding to the type, and in 32 bits two products, a sum and sines and cosines of at most 2 steps each
    assert ((heads[:, :H + G].double() - want).abs() <= torch.finfo(qkv.dtype).eps / 2 * want.abs() + 2 * mag * 2.0 ** -21).all()
    assert torch.equal(heads[:, H + G:], before.reshape(T, -1, D)[:, H + G:])
    # what is cached is the row as it now is: exactly its quantised form
    k_out, v_out = (torch.empty(T, G, D, dtype=qkv.dtype, device=DEV) for _ in range(2))
    ops.read_kv_fp8(*c.operands, pos, seq, slots, k_out, v_out)
    assert torch.equal(k_out.double().cpu(), plain.values(*plain.quantise(heads[:, H:H + G])))
    assert torch.equal(v_out.double().cpu(), plain.values(*plain.quantise(heads[:, H + G:])))


def test_rotation_without_a_write_leaves_the_cache():
    c = Cache([20], 1, 64, 16, 6)
    pos, seq, slots = step([(4, 10)], c.slots)
    qkv = rows(4, 2, 1, 64, torch.bfloat16, 7)
    inv = (10000.0 ** (-torch.arange(32).float() / 32)).to(DEV)
    before = [(p.view(torch.uint8).clone(), e.clone()) for p, e in c.dev]
    x = qkv.clone()
    ops.rope_kv_write_fp8(x, pos, seq, slots, inv, 64, *c.operands, 2, 1, 64, write_cache=False)
    y = qkv.clone()
    ops.rope_kv_write_fp8(y, pos, seq, slots, inv, 64, *c.operands, 2, 1, 64)
    assert torch.equal(x, y) and not torch.equal(x, qkv)
    z = [(p.view(torch.uint8), e) for p, e in c.dev]
    assert not torch.equal(z[0][0], before[0][0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,rot", [(64, 64), (20, 8)])
def test_no_byte_is_written_without_a_write(dtype, D, rot):
    c = Cache([20], 2, D, 16, 6)
    pos, seq, slots = step([(4, 10)], c.slots)
    qkv = rows(4, 2, 2, D, DTYPES[dtype], 7)
    inv, was = (10000.0 ** (-torch.arange(rot // 2).float() / (rot // 2))).to(DEV), qkv.clone()
    before = [(p.view(torch.uint8).clone(), e.clone()) for p, e in c.dev]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_kv_write_fp8(qkv, pos, seq, slots, inv, rot, *c.operands, 2, 2, D, write_cache=False, status=status)
    assert not torch.equal(qkv[:, :4 * D], was[:, :4 * D]) and torch.equal(qkv[:, 4 * D:], was[:, 4 * D:]) and int(status) == 0
    assert all(torch.equal(p.view(torch.uint8), p0) and torch.equal(e, e0) for (p, e), (p0, e0) in zip(c.dev, before))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_at_the_ends_of_the_range(dtype):
    G, D, P = 1, 64, 16
    c = Cache([P], G, D, P, 8)
    pos, seq, slots = step([(P, 0)], c.slots)
    qkv = torch.zeros(P, 3 * D, dtype=DTYPES[dtype], device=DEV)
    big = torch.finfo(qkv.dtype).max
    for i, (x, y) in enumerate([(0.0, 0.0), (448.0, -448.0), (449.0, 1.0), (big, -big), (big, 1e-3), (1e-38, -2e-39), (1e-40, 0.0), (math.nan, 1.0),
                                (math.inf, 1.0), (-math.inf, math.nan), (-0.0, 2.0 ** -9), (240.0, 15.5), (2.0 ** -119, 2.0 ** -128), (3.2e38, 3.3e38)]):
        qkv[i, D:2 * D:2], qkv[i, D + 1:2 * D:2], qkv[i, 2 * D:], qkv[i, 2 * D + 5] = x, y, y, x
    ops.rope_kv_write_fp8(qkv, pos, seq, slots, None, 0, *c.operands, 1, G, D)
    k_out, v_out = (torch.empty(P, G, D, dtype=qkv.dtype, device=DEV) for _ in range(2))
    ops.read_kv_fp8(*c.operands, pos, seq, slots, k_out, v_out)
    for got, x in ((k_out, qkv[:, D:2 * D]), (v_out, qkv[:, 2 * D:])):
        want = plain.values(*plain.quantise(x.reshape(P, G, D).cpu()))
        assert torch.equal(torch.nan_to_num(got.double().cpu(), nan=1e300), torch.nan_to_num(want, nan=1e300))
    assert torch.isfinite(k_out[:7]).all() and torch.isnan(k_out[7:10]).all()


@pytest.mark.parametrize("what", ["no page", "page behind the pool", "position behind the table", "negative position", "slot behind the table", "negative slot"])
def test_positions_without_a_page(what):
    G, D, P = 2, 64, 16
    c = Cache([30, 30], G, D, P, 9)
    pos, seq, slots = step([(3, 10), (3, 10)], c.slots)
    row = int(c.slots[1])
    if what == "no page":
        c.table[row, 0] = -1
    elif what == "page behind the pool":
        c.table[row, 0] = c.dev[0][0].shape[0]
    elif what == "position behind the table":
        pos[3:] = c.table.shape[1] * P + torch.arange(3, device=DEV)
    elif what == "negative position":
        pos[3:] = -1 - torch.arange(3, device=DEV)
    else:
        slots[1] = c.table.shape[0] if what.startswith("slot") else -1
    qkv = rows(6, 2, G, D, torch.bfloat16, 10)
    before = [(p.view(torch.uint8).clone(), e.clone()) for p, e in c.dev]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.rope_kv_write_fp8(qkv, pos, seq, slots, None, 0, *c.operands, 2, G, D, status=status)
    assert int(status) == 2
    page = int(c.table[int(c.slots[0]), 0])
    for (p, e), (p0, e0) in zip(c.dev, before):
        p = p.view(torch.uint8).clone()
        assert not torch.equal(p[page], p0[page])
        p[page, :, 10:13] = p0[page, :, 10:13]
        assert torch.equal(p, p0)
    k_out, v_out = (torch.full((6, G, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.read_kv_fp8(*c.operands, pos, seq, slots, k_out, v_out)
    assert (k_out[3:] == 0).all() and (v_out[3:] == 0).all() and (k_out[:3] != 0).any()
    # attention: the request with nothing to see gets zeros, the other one its result
    out = torch.full((6, 2 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    if what not in ("position behind the table",):
        ops.decode_attention_fp8(qkv, *c.operands, pos, seq, slots, out, 2, G, D, None, 0.1)
        assert (out[3:] == 0).all() and (out[:3] != 0).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("G,D,P,R", [(2, 64, 16, 16), (1, 128, 64, 64), (3, 20, 5, 5), (1, 256, 32, 32), (2, 128, 16, 128), (1, 48, 5, 128), (1, 64, 128, 16)])
def test_stretches_of_requests(dtype, G, D, P, R):
    lens = [5 * P - 1, 1, 3 * P, 2 * P + 1]
    c = Cache(lens, G, D, P, 11)
    c.table[int(c.slots[2]), 1] = -1                                        # a page in the middle is missing
    spans, row = [], 0
    for b, p0, end in [(0, 2 * P, lens[0]), (1, 0, 1), (2, 0, lens[2]), (3, P, 2 * P)]:
        spans.append((b, p0, end, row))
        row += -(-(end - p0) // R) * R
    k_out, v_out = (torch.full((row // R, G, R, D), 7.0, dtype=DTYPES[dtype], device=DEV) for _ in range(2))
    ops.read_kv_fp8_spans(*c.operands, torch.tensor(spans, dtype=torch.int32, device=DEV), row, c.slots.to(DEV), k_out, v_out)
    for which, got in ((0, k_out), (1, v_out)):
        want = torch.zeros(row, G, D, dtype=torch.float64)
        for b, p0, end, r in spans:
            x, there = c.of(b, end, which)
            want[r:r + end - p0] = torch.where(there[:, None, None], x, 0.0)[p0:]
        assert torch.equal(got.double().cpu().transpose(1, 2).reshape(row, G, D), want)


def test_nothing_to_do():
    c = Cache([4], 1, 64, 16, 12)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    qkv, out = rows(0, 2, 1, 64, torch.bfloat16, 1), torch.zeros(0, 128, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device=DEV)
    ops.rope_kv_write_fp8(qkv, none, none, c.slots.to(DEV), None, 0, *c.operands, 2, 1, 64)
    ops.read_kv_fp8(*c.operands, none, none, c.slots.to(DEV), k, k.clone())
    ops.decode_attention_fp8(qkv, *c.operands, none, none, c.slots.to(DEV), out, 2, 1, 64, None, 1.0)
    ops.prefill_attention_fp8(qkv, *c.operands, ops.prefill_fp8_plan([], 16, DEV), none, none, c.slots.to(DEV), out, 2, 1, 64, None, 1.0)


# ---- attention of few tokens ----------------------------------------------------------------------------------------
# what a weight is rounded to: in the decode kernels 2^-11 (16-bit rows: f16 in three parts of e4m3) or nothing to speak of
WEIGHT = {"bf16": 2.0 ** -10, "f32": 2.0 ** -20}
SHAPES = [(4, 2, 128, 16), (16, 16, 128, 64), (28, 4, 128, 64), (32, 2, 128, 128), (3, 3, 64, 48), (20, 1, 64, 16), (6, 3, 48, 32), (5, 1, 256, 64),
          (2, 2, 16, 16), (8, 8, 80, 16), (4, 2, 20, 16), (4, 2, 64, 5), (7, 1, 200, 7)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", SHAPES)
def test_decode(dtype, H, G, D, P):
    lens = [1, 2, P, P + 1, 127, 128, 129, 300]
    c = Cache(lens, G, D, P, H + D)
    entries = [(1, n - 1) for n in lens]
    q = rows(len(lens), H, G, D, DTYPES[dtype], 3)
    out = torch.full((len(lens), H * D), 7.0, dtype=q.dtype, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, None, D ** -0.5, status=status)
    assert int(status) == 0
    check(out, c, entries, q, H, None, D ** -0.5, None, WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 144, 16), (3, 1, 192, 32), (18, 2, 240, 64), (9, 1, 32, 48), (2, 2, 112, 80), (12, 1, 128, 16)])
@pytest.mark.parametrize("window", [None, 70])
def test_decode_of_other_head_sizes(dtype, H, G, D, P, window):
    """Heads that end inside a slab of 128 elements or a step of 32, pages that hold no whole tile; a row named twice."""
    lens = [1, 63, 128, 500, 1300]
    c = Cache(lens, G, D, P, H + D + 1)
    entries = [(1, n - 1) for n in lens]
    q, st = rows(5, H, G, D, DTYPES[dtype], 5, extra=3), step(entries, c.slots)
    out = torch.full((5, H * D + 1), 7.0, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *st, out[:, :H * D], H, G, D, window, D ** -0.5, softcap=30.0)
    check(out[:, :H * D], c, entries, q, H, window, D ** -0.5, 30.0, WEIGHT[dtype])
    some = torch.full_like(out, 7.0)
    ops.decode_attention_fp8(q, *c.operands, *st, some[:, :H * D], H, G, D, window, D ** -0.5, softcap=30.0,
                             tokens=torch.tensor([4, 0, 4, 3, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(some[[0, 3, 4]], out[[0, 3, 4]]) and (some[[1, 2]] == 7).all() and (out[:, H * D:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 5000])
@pytest.mark.parametrize("softcap", [None, 5.0])
def test_decode_with_a_window(dtype, window, softcap):
    H, G, D, P = 6, 2, 64, 16
    lens = [1, 60, 129, 400, 1000]
    c = Cache(lens, G, D, P, window)
    entries = [(1, n - 1) for n in lens]
    q = rows(len(lens), H, G, D, DTYPES[dtype], 4, extra=5)
    out = torch.empty(len(lens), H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, window, 0.3, softcap=softcap)
    check(out, c, entries, q, H, window, 0.3, softcap, WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 128, 64), (7, 1, 64, 16), (4, 4, 256, 32)])
def test_several_tokens_a_request_and_some_rows_only(dtype, H, G, D, P):
    lens = [20, 333, 8]
    c = Cache(lens, G, D, P, 5)
    entries = [(5, 15), (8, 325), (8, 0)]
    q = rows(21, H, G, D, DTYPES[dtype], 6)
    out = torch.full((21, H * D + 8), 7.0, dtype=q.dtype, device=DEV)
    st = step(entries, c.slots)
    ops.decode_attention_fp8(q, *c.operands, *st, out[:, :H * D], H, G, D, None, 0.1)
    assert (out[:, H * D:] == 7).all()
    check(out[:, :H * D], c, entries, q, H, None, 0.1, None, WEIGHT[dtype])
    some = torch.full_like(out, 7.0)
    at = torch.tensor([20, 0, 7], dtype=torch.int32, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *st, some[:, :H * D], H, G, D, None, 0.1, tokens=at)
    assert torch.equal(some[at.long()], out[at.long()])
    some[at.long()] = 7
    assert (some == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("spread,q_scale", [(3.0, 1.0), (12.0, 1.0), (0.0, 30.0), (0.0, 1e-6)])
def test_rows_of_unequal_size(dtype, spread, q_scale):
    """Scales over many powers of two; sharp and flat distributions."""
    H, G, D, P = 4, 2, 64, 16
    lens = [700, 50]
    c = Cache(lens, G, D, P, 7, spread=spread)
    entries = [(1, n - 1) for n in lens]
    q = rows(2, H, G, D, DTYPES[dtype], 8, q_scale=q_scale / max(1.0, 4 ** spread if spread < 5 else 1e9))
    out = torch.empty(2, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, None, 0.125)
    check(out, c, entries, q, H, None, 0.125, None, WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_long_context(dtype):
    H, G, D, P = 4, 1, 128, 64
    lens = [20011, 64, 9000]
    c = Cache(lens, G, D, P, 9)
    entries = [(1, n - 1) for n in lens]
    q = rows(3, H, G, D, DTYPES[dtype], 10)
    out = torch.empty(3, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, None, D ** -0.5)
    check(out, c, entries, q, H, None, D ** -0.5, None, WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets_past_32_bits(dtype):
    """A pool of which the last pages' elements lie past 2^32."""
    H, G, D, P = 4, 4, 256, 128
    c = Cache([200, 70], G, D, P, 10, pool=(1 << 32) // (G * P * D) + 5)
    entries = [(1, 199), (1, 69)]
    q = rows(2, H, G, D, DTYPES[dtype], 11)
    st = step(entries, c.slots)
    ops.rope_kv_write_fp8(q, *st, None, 0, *c.operands, H, G, D)
    k, v = (torch.empty(2, G, D, dtype=q.dtype, device=DEV) for _ in range(2))
    ops.read_kv_fp8(*c.operands, *st, k, v)
    assert torch.equal(k.double().cpu(), plain.values(*plain.quantise(q[:, H * D:(H + G) * D].reshape(2, G, D).cpu())))
    out = torch.empty(2, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, 0.05)
    check(out, c, entries, q, H, None, 0.05, None, WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D,P", [(64, 16), (20, 5)])
def test_rows_that_are_no_numbers_reach_who_sees_them(dtype, D, P):
    H, G = 4, 2
    lens = [50, 50, 50, 50, 300]
    c = Cache(lens, G, D, P, 13)
    for b, where, which in ((0, 49, 0), (1, 20, 1), (3, 3, 0), (4, 150, 1)):       # requests 3 and 4: outside the window
        page = int(c.table[int(c.slots[b]), where // P])
        c.dev[which][1][page, 1, where % P] = 255
    c.dev[1][1][int(c.table[int(c.slots[2]), 49 // P]), :, 49 % P] = 255           # request 2's last position: not seen from 48
    entries = [(1, 49), (1, 49), (1, 48), (1, 49), (1, 299)]
    q = rows(5, H, G, D, DTYPES[dtype], 12)
    out = torch.empty(5, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, 40, 0.1)
    check(out, c, entries, q, H, 40, 0.1, None, WEIGHT[dtype])
    bad = torch.isnan(out).reshape(5, H, D).any(-1).cpu()
    assert bad.tolist() == [[False, False, True, True]] * 2 + [[False] * 4] * 3
    q[1, D] = math.nan
    q[3, 0] = math.inf
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, 40, 0.1)
    bad = torch.isnan(out).reshape(5, H, D).all(-1).cpu()
    assert bad.tolist() == [[False, False, True, True], [False, True, True, True], [False] * 4, [True, False, False, False], [False] * 4]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_missing_pages_do_not_count(dtype):
    H, G, D, P = 4, 2, 64, 16
    c = Cache([200, 200], G, D, P, 14)
    c.table[int(c.slots[0]), 3:9] = -1
    c.table[int(c.slots[1]), :] = -1
    entries = [(1, 199), (1, 199)]
    q = rows(2, H, G, D, DTYPES[dtype], 15)
    out = torch.full((2, H * D), 7.0, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, None, 0.1)
    check(out, c, entries, q, H, None, 0.1, None, WEIGHT[dtype])
    assert (out[1] == 0).all()


# ---- attention of prompt portions -----------------------------------------------------------------------------------
# weights are rounded to bfloat16 before the second product (half a step: 2^-8 of the weight), in 32 bits to three parts of it
PROMPT_WEIGHT = {"bf16": 2.0 ** -8, "f32": 2.0 ** -20}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 128, 64), (4, 4, 64, 64), (6, 3, 48, 32), (2, 1, 128, 16), (5, 1, 256, 64), (4, 2, 20, 16), (2, 2, 128, 5), (8, 8, 80, 128),
                                     (7, 1, 128, 64), (28, 4, 64, 16), (130, 2, 16, 64), (129, 1, 32, 16), (128, 1, 64, 5), (12, 4, 112, 64)])
def test_prompts(dtype, H, G, D, P):
    entries = [(9, 0), (1, 40), (70, 0), (8, 3), (33, 100), (130, 17)]
    c = Cache([n + s for n, s in entries], G, D, P, 16)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, DTYPES[dtype], 17)
    out = torch.empty(T, H * D, dtype=q.dtype, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *step(entries, c.slots), out, H, G, D, None, D ** -0.5,
                              status=status)
    assert int(status) == 0
    check(out, c, entries, q, H, None, D ** -0.5, None, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,softcap", [(1, None), (50, None), (64, 5.0), (None, 5.0), (1000, 30.0)])
@pytest.mark.parametrize("most", [1, 1 << 30])
def test_prompts_with_a_window(dtype, window, softcap, most, monkeypatch):
    monkeypatch.setattr(ops, "FP8_READ_BACK_MAX", most)
    H, G, D, P = 4, 2, 64, 64
    entries = [(120, 0), (300, 200), (2, 9), (15, 64)]
    c = Cache([n + s for n, s in entries], G, D, P, 18)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, DTYPES[dtype], 19)
    out = torch.empty(T, H * D, dtype=q.dtype, device=DEV)
    plan = ops.prefill_fp8_plan(entries, P, DEV)
    for _ in range(2):                                                      # (a plan serves every layer of a step)
        out.fill_(7.0)
        ops.prefill_attention_fp8(q, *c.operands, plan, *step(entries, c.slots), out, H, G, D, window, 0.2, softcap=softcap)
        check(out, c, entries, q, H, window, 0.2, softcap, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("dtype,H,softcap", [("bf16", 2, None), ("bf16", 1, None), ("bf16", 2, 20.0), ("f32", 2, None)])
@pytest.mark.parametrize("D", [64, 256])
def test_a_prompt_next_to_rows_that_are_no_numbers(dtype, H, softcap, D):
    """Garbage behind a request's last position, and a row that only some queries see; heads that share their keys, and one that
    does not."""
    G, P = 1, 64
    entries = [(100, 0), (90, 30)]
    c = Cache([170, 128], G, D, P, 20)
    for which in (0, 1):
        c.dev[which][1][int(c.table[int(c.slots[0]), 1]), :, 100 - P:] = 255
        c.dev[which][1][int(c.table[int(c.slots[1]), 1]), :, 120 - P:] = 255
    c.dev[1][1][int(c.table[int(c.slots[0]), 0]), :, 60] = 255
    T = 190
    q = rows(T, H, G, D, DTYPES[dtype], 21)
    out = torch.empty(T, H * D, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *step(entries, c.slots), out, H, G, D, None, 0.1, softcap=softcap)
    bad = torch.isnan(out).any(-1).cpu()
    assert bad[:60].sum() == 0 and bad[60:100].all() and not bad[100:].any()
    assert torch.isfinite(out[:60]).all() and torch.isfinite(out[100:]).all()


@pytest.mark.parametrize("dtype,H,G,D,extra", [("bf16", 4, 2, 64, 2), ("bf16", 2, 2, 128, 2), ("bf16", 4, 1, 256, 2), ("bf16", 129, 1, 32, 0), ("bf16", 130, 1, 144, 0),
                                               ("f32", 4, 2, 20, 0), ("f32", 3, 1, 68, 0), ("f32", 4, 2, 64, 1), ("f32", 2, 2, 128, 0)])
@pytest.mark.parametrize("window,softcap", [(None, None), (25, None), (None, 20.0)])
def test_rows_that_are_no_numbers_by_every_route(dtype, H, G, D, extra, window, softcap):
    """Results off the 16-byte grid, more query heads a kv head than a tile has rows, odd head sizes: who sees such a row, and nobody else."""
    entries = [(100, 0), (70, 30), (9, 4)]
    c = Cache([100, 128, 13], G, D, 64, 100)
    for b, at, which in ((0, 60, 1), (0, 99, 0), (1, 20, 0), (1, 29, 1), (1, 120, 0)):      # (behind 120, 20 and 29: in the window of some)
        c.dev[which][1][int(c.table[int(c.slots[b]), at // 64]), :, at % 64] = 255
    T = 179
    q = rows(T, H, G, D, DTYPES[dtype], 101)
    out = torch.full((T, H * D + extra), 7.0, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *step(entries, c.slots), out[:, :H * D], H, G, D, window, 0.1, softcap=softcap)
    check(out[:, :H * D], c, entries, q, H, window, 0.1, softcap, PROMPT_WEIGHT[dtype])
    assert (out[:, H * D:] == 7).all()


@pytest.mark.parametrize("H,G,D", [(6, 2, 128), (7, 1, 64), (16, 4, 80), (6, 2, 256), (5, 1, 144)])
@pytest.mark.parametrize("window", [None, 100, 700])
@pytest.mark.parametrize("run_blocks", [0, 1, 3])
@pytest.mark.parametrize("softcap", [None, 6.0])
def test_prompts_of_grouped_heads_cut_into_runs(H, G, D, window, run_blocks, softcap, monkeypatch):
    own = ops.prefill_tc_plan
    monkeypatch.setattr(ops, "prefill_tc_plan", lambda *a, **k: own(*a, run_blocks=run_blocks, **k))
    entries = [(60, 900), (300, 0), (19, 333)]
    c = Cache([n + s for n, s in entries], G, D, 64, 50)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, torch.bfloat16, 51)
    out = torch.full((T, H * D), 7.0, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *step(entries, c.slots), out, H, G, D, window, 0.15, softcap=softcap)
    check(out, c, entries, q, H, window, 0.15, softcap, PROMPT_WEIGHT["bf16"])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (2, 2, 256)])
@pytest.mark.parametrize("entries", [[(12, 100), (9, 3)], [(1, 200), (1, 7), (30, 0), (3, 50), (400, 100), (1, 90)]])
def test_prompts_as_chosen(dtype, H, G, D, entries, monkeypatch):
    """Tokens one by one where that is sooner, portions with single tokens between them where it is not."""
    monkeypatch.setattr(ops, "fp8_token_by_token", CHOICE)
    c = Cache([n + s for n, s in entries], G, D, 64, 83)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, DTYPES[dtype], 84)
    for window in (None, 33):
        out = torch.full((T, H * D), 7.0, dtype=q.dtype, device=DEV)
        ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *step(entries, c.slots), out, H, G, D, window, 0.15)
        check(out, c, entries, q, H, window, 0.15, None, PROMPT_WEIGHT[dtype])


def test_results_beside_a_portion_stay():
    """Rows of a wider result behind a head's, and a tile's places that no token has, are left as they were."""
    H, G, D = 6, 2, 64
    entries = [(50, 0), (23, 70)]
    c = Cache([50, 93], G, D, 64, 52)
    q = rows(73, H, G, D, torch.bfloat16, 53)
    out = torch.full((75, H * D + 8), 7.0, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *step(entries, c.slots), out[:73, :H * D], H, G, D, None, 0.1)
    assert (out[73:] == 7).all() and (out[:, H * D:] == 7).all()
    check(out[:73, :H * D], c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT["bf16"])


def only_seen(c, entries, window):
    """Everything in the cache but what the entries' tokens see becomes bytes that are no numbers, with exponents of any kind."""
    g = torch.Generator().manual_seed(60)
    keep = torch.zeros(c.dev[0][0].shape[0], c.P, dtype=torch.bool)
    for b, (n, start) in enumerate(entries):
        for p in range(max(0, start - window + 1) if window else 0, start + n):
            keep[int(c.table[int(c.slots[b]), p // c.P]), p % c.P] = True
    keep = keep[:, None].expand(-1, c.G, -1)
    for i, (pages, e) in enumerate(c.dev):
        bad = torch.where(torch.rand(pages.shape, generator=g) < 0.5, 127, 255).to(torch.uint8)
        pages = torch.where(keep[..., None], pages.view(torch.uint8).cpu(), bad).to(DEV).view(torch.float8_e4m3fn)
        c.dev[i] = (pages, torch.where(keep, e.cpu(), torch.randint(8, 256, e.shape, generator=g).to(torch.uint8)).to(DEV))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 128, 64), (6, 2, 64, 16), (4, 1, 256, 128), (2, 2, 20, 5), (1, 1, 64, 48)])
@pytest.mark.parametrize("window", [None, 37])
def test_what_nobody_has_written_counts_for_nothing(dtype, H, G, D, P, window):
    lens = [1, 5, 127, 130, 400]
    c = Cache(lens, G, D, P, 61)
    entries = [(1, n - 1) for n in lens]
    only_seen(c, entries, window)
    q = rows(len(lens), H, G, D, DTYPES[dtype], 62)
    out = torch.empty(len(lens), H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, window, 0.1)
    check(out, c, entries, q, H, window, 0.1, None, WEIGHT[dtype])
    entries = [(1, 0), (5, 0), (60, 67), (2, 128), (40, 360)]
    c = Cache(lens, G, D, P, 63)
    only_seen(c, entries, window)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, DTYPES[dtype], 64)
    out = torch.empty(T, H * D, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *step(entries, c.slots), out, H, G, D, window, 0.1)
    check(out, c, entries, q, H, window, 0.1, None, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("R,P", [(128, 64), (64, 64), (16, 5)])
def test_stretches_that_begin_inside_a_page(R, P):
    G, D = 2, 64
    c = Cache([300, 200], G, D, P, 65)
    spans, row = [], 0
    for b, p0, end in [(0, 130, 300), (1, 64, 200), (0, 7, 9)]:
        spans.append((b, p0, end, row + p0 % R))
        row += (-(-end // R) - p0 // R) * R
    k, v = (torch.full((row // R, G, R, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    ops.read_kv_fp8_spans(*c.operands, torch.tensor(spans, dtype=torch.int32, device=DEV), row, c.slots.to(DEV), k, v)
    for which, got in ((0, k), (1, v)):
        want = torch.zeros(row, G, D, dtype=torch.float64)
        for b, p0, end, r in spans:
            want[r:r + end - p0] = c.of(b, end, which)[0][p0:]
        assert torch.equal(got.double().cpu().transpose(1, 2).reshape(row, G, D), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("softcap", [None, 4.0])
def test_scales_that_are_not_positive(dtype, scale, softcap):
    H, G, D, P = 4, 2, 64, 64
    entries = [(1, 149), (40, 60), (12, 0)]
    c = Cache([150, 100, 12], G, D, P, 74)
    q = rows(53, H, G, D, DTYPES[dtype], 75)
    st, out = step(entries, c.slots), torch.empty(53, H * D, dtype=DTYPES[dtype], device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, scale, softcap=softcap)
    check(out, c, entries, q, H, None, scale, softcap, WEIGHT[dtype])
    out.fill_(7.0)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *st, out, H, G, D, None, scale, softcap=softcap)
    check(out, c, entries, q, H, None, scale, softcap, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [1e-50, 1e-40, 2.0 ** -126])
@pytest.mark.parametrize("softcap", [None, 4.0])
def test_scales_that_32_bits_hardly_hold(dtype, scale, softcap):
    """All keys that are seen count the same then."""
    H, G, D, P = 4, 2, 64, 64
    entries = [(40, 60), (120, 0)]
    c = Cache([100, 120], G, D, P, 98)
    q = rows(160, H, G, D, DTYPES[dtype], 99)
    st, out = step(entries, c.slots), torch.full((160, H * D), 7.0, dtype=DTYPES[dtype], device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *st, out, H, G, D, None, scale, softcap=softcap)
    check(out, c, entries, q, H, None, scale, softcap, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 128, 256), (3, 1, 64, 384), (2, 2, 20, 1), (2, 1, 256, 512), (8, 1, 16, 1024)])
def test_pages_longer_than_a_tile(dtype, H, G, D, P):
    lens = [1, 100, 700, 1500]
    c = Cache(lens, G, D, P, 76)
    entries = [(1, n - 1) for n in lens]
    q = rows(4, H, G, D, DTYPES[dtype], 77)
    st, out = step(entries, c.slots), torch.empty(4, H * D, dtype=DTYPES[dtype], device=DEV)
    ops.rope_kv_write_fp8(q, *st, None, 0, *c.operands, H, G, D)
    ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, 0.1)
    check(out, c, entries, q, H, None, 0.1, None, WEIGHT[dtype])
    entries = [(1, 0), (50, 50), (300, 400), (20, 1480)]
    q = rows(371, H, G, D, DTYPES[dtype], 78)
    out = torch.empty(371, H * D, dtype=DTYPES[dtype], device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *step(entries, c.slots), out, H, G, D, None, 0.1)
    check(out, c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT[dtype])


@pytest.mark.parametrize("H,G,D", [(4, 4, 128), (3, 3, 48), (12, 12, 64), (2, 2, 256), (3, 3, 192)])
@pytest.mark.parametrize("window,softcap", [(None, None), (90, None), (90, 40.0)])
def test_prompts_of_heads_with_their_own_keys(H, G, D, window, softcap):
    """Portions around the sizes of a sub-tile and a tile."""
    entries = [(127, 0), (128, 5), (129, 0), (256, 131), (257, 0), (9, 300)]
    c = Cache([n + s for n, s in entries], G, D, 64, 79)
    T = sum(n for n, _ in entries)
    q = rows(T, H, G, D, torch.bfloat16, 80)
    out = torch.full((T, H * D), 7.0, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *step(entries, c.slots), out, H, G, D, window, 0.15, softcap=softcap)
    check(out, c, entries, q, H, window, 0.15, softcap, PROMPT_WEIGHT["bf16"])


@pytest.mark.parametrize("first,second", [((8, 8, 64, "bf16"), (8, 8, 128, "bf16")), ((8, 8, 128, "bf16"), (8, 8, 64, "bf16")), ((8, 2, 64, "f32"), (8, 8, 64, "f32")),
                                          ((8, 8, 64, "f32"), (8, 2, 64, "f32")), ((4, 1, 256, "bf16"), (4, 4, 256, "bf16")), ((4, 4, 64, "f32"), (4, 4, 64, "bf16"))])
def test_a_plan_of_layers_that_are_cut_differently(first, second, monkeypatch):
    """Layers whose steps are cut into other portions, by what they read back of a position, use one plan in turn: every result is that of
    a plan of the layer's own, bit for bit."""
    monkeypatch.setattr(ops, "FP8_READ_BACK_MAX", 1 << 20)
    entries = [(40, 460), (12, 100), (3, 90), (100, 20), (30, 300), (20, 0)]
    plan, cuts = ops.prefill_fp8_plan(entries, 64, DEV), []
    for H, G, D, dtype in (first, second, first):
        c = Cache([n + s for n, s in entries], G, D, 64, 90)
        T = sum(n for n, _ in entries)
        q, st, own = rows(T, H, G, D, DTYPES[dtype], 91), step(entries, c.slots), ops.prefill_fp8_plan(entries, 64, DEV)
        want, out = (torch.full((T, H * D), 7.0, dtype=q.dtype, device=DEV) for _ in range(2))
        ops.prefill_attention_fp8(q, *c.operands, own, *st, want, H, G, D, None, 0.1)
        ops.prefill_attention_fp8(q, *c.operands, plan, *st, out, H, G, D, None, 0.1)
        assert torch.equal(out, want)
        cuts.append([n for _, n, *_ in own.parts(None, 2 * G * D * q.element_size())])
    assert cuts[0] != cuts[1] and cuts[0] == cuts[2]
    check(out, c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT[first[3]])


@pytest.mark.parametrize("softcap", [1e5, 1e6, 1e7, 1e30])
@pytest.mark.parametrize("dtype,H,G,D", [("bf16", 4, 2, 128), ("bf16", 3, 3, 64), ("bf16", 6, 2, 256), ("f32", 4, 2, 128)])
def test_caps_far_beyond_the_scores(dtype, H, G, D, softcap):
    """A capped score is exact in proportion to itself, not to its cap.  Against the definition without a cap: scores are below 32 in size,
    and c tanh(s / c) is off s by at most |s|^3 / (3 c^2), 1.1e-6 here and below what a score's own arithmetic may be off by."""
    entries = [(9, 0), (33, 2), (200, 70), (1, 90), (300, 0)]
    c = Cache([n + s for n, s in entries], G, D, 64, 92)
    T = sum(n for n, _ in entries)
    q, st = rows(T, H, G, D, DTYPES[dtype], 93), step(entries, c.slots)
    out = torch.full((T, H * D), 7.0, dtype=q.dtype, device=DEV)
    ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, 64, DEV), *st, out, H, G, D, None, D ** -0.5, softcap=softcap)
    check(out, c, entries, q, H, None, D ** -0.5, None, PROMPT_WEIGHT[dtype])
    ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, D ** -0.5, softcap=softcap)
    check(out, c, entries, q, H, None, D ** -0.5, None, WEIGHT[dtype])


@pytest.mark.parametrize("softcap", [0.3, 2.0])
@pytest.mark.parametrize("D", [64, 256])
def test_scores_on_either_side_of_half_the_cap(softcap, D):
    """Scores from far below the cap to far beyond it in one row, and a request's bits whatever the request beside it has: which of the
    two forms a score takes is its own affair."""
    H, G = 4, 2
    entries = [(70, 60), (150, 0)]
    c = Cache([130, 150], G, D, 64, 94)
    q = rows(220, H, G, D, torch.bfloat16, 95)
    q[:70] *= torch.exp2(torch.linspace(-12, 4, 70)).to(DEV)[:, None].bfloat16()
    st, plan, outs = step(entries, c.slots), ops.prefill_fp8_plan(entries, 64, DEV), []
    for size in (1.0, 0.0, 1000.0):
        x = q.clone()
        x[70:] *= size
        out = torch.full((220, H * D), 7.0, dtype=q.dtype, device=DEV)
        ops.prefill_attention_fp8(x, *c.operands, plan, *st, out, H, G, D, None, D ** -0.5, softcap=softcap)
        outs.append(out)
    check(outs[0], c, entries, q, H, None, D ** -0.5, softcap, PROMPT_WEIGHT["bf16"])
    assert torch.equal(outs[0][:70], outs[1][:70]) and torch.equal(outs[0][:70], outs[2][:70])


# ---- streams, graphs, order -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_on_a_stream_of_its_own_and_in_a_graph(dtype):
    H, G, D, P = 8, 2, 128, 64
    lens = [900, 70, 1, 2000]
    c = Cache(lens, G, D, P, 22)
    entries = [(1, n - 1) for n in lens]
    q = rows(4, H, G, D, DTYPES[dtype], 23)
    st, operands = step(entries, c.slots), c.operands
    want = torch.empty(4, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *operands, *st, want, H, G, D, None, 0.09)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.zeros_like(want)
    ops.decode_attention_fp8(q, *operands, *st, out, H, G, D, None, 0.09, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)
    # captured: replays follow what the buffers hold, and two graphs do not share what they need
    graphs, outs = [], [torch.zeros_like(want) for _ in range(2)]
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.rope_kv_write_fp8(q, *st, None, 0, *operands, H, G, D)
            ops.decode_attention_fp8(q, *operands, *st, o, H, G, D, None, 0.09)
        graphs.append(g)
    for seed in (24, 25):
        q.copy_(rows(4, H, G, D, DTYPES[dtype], seed))
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        for s, g in zip((a, b), graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        ops.decode_attention_fp8(q, *operands, *st, want, H, G, D, None, 0.09)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        check(want, c, entries, q, H, None, 0.09, None, WEIGHT[dtype])


def test_a_prompt_on_a_stream_of_its_own():
    H, G, D, P = 4, 2, 64, 64
    entries = [(300, 50), (9, 0)]
    c = Cache([350, 9], G, D, P, 26)
    q = rows(309, H, G, D, torch.bfloat16, 27)
    st, plan = step(entries, c.slots), ops.prefill_fp8_plan(entries, P, DEV)
    want, out = torch.empty(309, H * D, dtype=q.dtype, device=DEV), torch.zeros(309, H * D, dtype=q.dtype, device=DEV)
    operands = c.operands
    ops.prefill_attention_fp8(q, *operands, plan, *st, want, H, G, D, None, 0.1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ops.prefill_attention_fp8(q, *operands, plan, *st, out, H, G, D, None, 0.1, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)
    other = torch.zeros_like(out)
    with torch.cuda.stream(side):
        ops.prefill_attention_fp8(q, *operands, plan, *st, other, H, G, D, None, 0.1)
    side.synchronize()
    assert torch.equal(other, want)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_runs_on_a_stream_of_their_own(D):
    """The kernel over pages of 128 on a named stream that begins late: what its runs leave is not handed to the current stream meanwhile."""
    H, G, entries = 4, 2, [(50, 1200)]
    items, merges, parts = ops.prefill_tc_plan(entries, None, G, tile=(2 if D <= 128 else 1) * 64, run_blocks=2)
    assert parts > 1
    g = torch.Generator().manual_seed(97)
    q, k, v = (torch.randn(*shape, generator=g).bfloat16().to(DEV) for shape in ((50, H * D), (10, G, 128, D), (10, G, 128, D)))
    table, items, merges = torch.arange(10, dtype=torch.int32, device=DEV)[None], torch.from_numpy(items).to(DEV), torch.from_numpy(merges).to(DEV)
    args = (q, k, v, table, items)
    want, out = torch.zeros(50, H * D, dtype=q.dtype, device=DEV), torch.zeros(50, H * D, dtype=q.dtype, device=DEV)
    ops.prefill_attention_grouped(*args, want, H, G, D, None, 0.1, merges=merges, parts=parts)
    torch.cuda.synchronize()
    side, floats = torch.cuda.Stream(), parts * G * (256 if D <= 128 else 128) * (max(D, 64) + 2)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                                       # (some 10 ms)
    ops.prefill_attention_grouped(*args, out, H, G, D, None, 0.1, merges=merges, parts=parts, stream=side.cuda_stream)
    others = [torch.full((floats,), 3.0, device=DEV) for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(out, want) and all(bool((x == 3).all()) for x in others)


def test_the_default_stream_named_from_another():
    """Calls that name the default stream while another is current; a plan that goes from one to the other and back."""
    H, G, D, P = 4, 2, 64, 64
    entries = [(300, 50), (3, 1400)]
    c = Cache([350, 1403], G, D, P, 105)
    q = rows(303, H, G, D, torch.bfloat16, 106)
    st, plan, operands = step(entries, c.slots), ops.prefill_fp8_plan(entries, P, DEV), c.operands
    outs = [torch.zeros(303, H * D, dtype=q.dtype, device=DEV) for _ in range(6)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.prefill_attention_fp8(q, *operands, plan, *st, outs[0], H, G, D, None, 0.1, stream=0)
        ops.prefill_attention_fp8(q, *operands, plan, *st, outs[1], H, G, D, None, 0.1)
        ops.decode_attention_fp8(q, *operands, *st, outs[2], H, G, D, None, 0.1, stream=0)
        ops.decode_attention_fp8(q, *operands, *st, outs[3], H, G, D, None, 0.1)
    ops.prefill_attention_fp8(q, *operands, plan, *st, outs[4], H, G, D, None, 0.1)
    ops.prefill_attention_fp8(q, *operands, plan, *st, outs[5], H, G, D, None, 0.1, stream=side.cuda_stream)
    torch.cuda.synchronize()
    check(outs[0], c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT["bf16"])
    check(outs[2], c, entries, q, H, None, 0.1, None, WEIGHT["bf16"])
    assert all(torch.equal(outs[0], outs[i]) for i in (1, 4, 5)) and torch.equal(outs[2], outs[3])


@pytest.mark.parametrize("first_named", [False, True])
def test_a_plan_made_on_a_default_stream_that_is_late(first_named):
    """Another stream's use of a plan waits for the lists, which the default stream has still to copy."""
    H, G, D, P = 4, 2, 64, 64
    entries = [(300, 50), (40, 1400), (200, 0)]
    c = Cache([350, 1440, 200], G, D, P, 107)
    q = rows(540, H, G, D, torch.bfloat16, 108)
    st, plan, operands = step(entries, c.slots), ops.prefill_fp8_plan(entries, P, DEV), c.operands
    late, out = (torch.zeros(540, H * D, dtype=q.dtype, device=DEV) for _ in range(2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert ops._stream_of(0, 0) == torch.cuda.default_stream(0) and ops._stream_of(side.cuda_stream, 0).cuda_stream == side.cuda_stream
    torch.cuda._sleep(40_000_000)                                           # (some 20 ms)
    with torch.cuda.stream(side if first_named else torch.cuda.default_stream()):
        ops.prefill_attention_fp8(q, *operands, plan, *st, late, H, G, D, None, 0.1, stream=0)
    with torch.cuda.stream(side):
        ops.prefill_attention_fp8(q, *operands, plan, *st, out, H, G, D, None, 0.1)
    torch.cuda.synchronize()
    check(out, c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT["bf16"])
    assert torch.equal(late, out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_request_has_the_same_bits_alone_and_twice(dtype):
    """The order of a token's sums depends on the step's size and the table's width only."""
    H, G, D, P = 16, 4, 128, 64
    c = Cache([1500] * 8, G, D, P, 28)
    entries = [(1, 1499)] * 8
    q = rows(1, H, G, D, DTYPES[dtype], 29).expand(8, -1).contiguous()
    for b in range(1, 8):
        c.table[int(c.slots[b])] = c.table[int(c.slots[0])]
    outs = []
    for _ in range(3):
        out = torch.empty(8, H * D, dtype=q.dtype, device=DEV)
        ops.decode_attention_fp8(q, *c.operands, *step(entries, c.slots), out, H, G, D, None, 0.09)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs) and all(torch.equal(outs[0][b], outs[0][0]) for b in range(8))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [None, 200])
def test_single_tokens_have_their_bits_whoever_is_beside_them(dtype, window):
    """In a step of as many tokens over a table as wide, a request's results do not hang on the other requests' lengths or places."""
    H, G, D, P, outs = 16, 4, 128, 64, []
    for others in ([1500] * 7, [1, 40, 128, 129, 700, 1400, 1500], [1] * 7):
        for place in (0, 5):
            c = Cache([1500] * 8, G, D, P, 102)
            lens = others[:place] + [1333] + others[place:]
            slots = torch.cat([c.slots[1:1 + place], c.slots[:1], c.slots[1 + place:]])
            q = rows(8, H, G, D, DTYPES[dtype], 103 + place)
            q[place] = rows(1, H, G, D, DTYPES[dtype], 104)[0]
            out = torch.empty(8, H * D, dtype=q.dtype, device=DEV)
            ops.decode_attention_fp8(q, *c.operands, *step([(1, n - 1) for n in lens], slots), out, H, G, D, window, 0.09)
            outs.append(out[place])
    assert all(torch.equal(o, outs[0]) for o in outs)


# ---- the operators as an engine uses them ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_request_from_prompt_to_tokens(dtype):
    """Two portions of a prompt and then single tokens, through write, prompt and decode attention, against attention over the
    quantised rows."""
    H, G, D, P = 4, 2, 64, 16
    c = Cache([120, 64], G, D, P, 30)
    done = [0, 0]
    for news in ([40, 20], [50, 9], [1, 1], [1, 1], [1, 2]):
        entries = [(n, d) for n, d in zip(news, done)]
        T = sum(news)
        q = rows(T, H, G, D, DTYPES[dtype], 31 + sum(done))
        st = step(entries, c.slots)
        ops.rope_kv_write_fp8(q, *st, None, 0, *c.operands, H, G, D)
        out = torch.empty(T, H * D, dtype=q.dtype, device=DEV)
        if max(news) > ops.FP8_FEW_TOKENS:
            ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan(entries, P, DEV), *st, out, H, G, D, None, 0.125)
        else:
            ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, 0.125)
        check(out, c, entries, q, H, None, 0.125, None, PROMPT_WEIGHT[dtype])
        done = [d + n for d, n in zip(done, news)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_operands_are_found_the_same_without_the_extension(dtype, monkeypatch):
    """What the extension module says of a call's tensors is what the plain look at them says, and what it does not take is
    refused by the plain one."""
    H, G, D, P = 4, 2, 64, 16
    c = Cache([70, 9, 33], G, D, P, 40)
    q = rows(3, H, G, D, DTYPES[dtype], 41, extra=8)
    st = step([(1, 69), (1, 8), (1, 32)], c.slots)
    out = torch.zeros(3, H * D + 4, dtype=q.dtype, device=DEV)
    k, v, ke, ve, table, _ = c.operands
    status, some = torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([2, 0], dtype=torch.int32, device=DEV)
    assert ops._look()("iT", st[0]) is not None                            # (it is there at all)
    for tensors in ([k, v, ke, ve, table, *st, q, out, status, some], [k, v, ke, ve, table, *st, q[:1].expand(3, -1), out[:, :H * D], None, None],
                    [k, v, ke, ve, table, *st, q[::2].repeat(2, 1)[:3], out, status, some[:0]]):
        labels = ops._CACHE_FP8 + ops._STEP + ("q", "out", "status", "tokens")
        assert ops._operands("x", ops._ATTEND_FP8, labels, *tensors) == ops._operands_slowly("x", ops._ATTEND_FP8, labels, tensors)
    for at, bad in ((0, k.view(torch.uint8)), (1, v[:1]), (2, ke.float()), (4, table.long()), (5, st[0][:2]), (8, q.double()), (8, q.T), (9, out.to(torch.float16)),
                    (0, k.transpose(1, 2)), (6, st[1].cpu()), (9, out[:, ::2]), (8, None)):
        t = [k, v, ke, ve, table, *st, q, out, status, some]
        t[at] = bad
        assert ops._look()(ops._ATTEND_FP8, *t) is None
        with pytest.raises(ops.KernelError):
            ops._operands("x", ops._ATTEND_FP8, ops._CACHE_FP8 + ops._STEP + ("q", "out", "status", "tokens"), *t)
    want = torch.empty(3, H * D, dtype=q.dtype, device=DEV)
    ops.decode_attention_fp8(q, *c.operands, *st, want, H, G, D, 40, 0.1)
    monkeypatch.setattr(ops, "_look", lambda: lambda *a: None)
    got = torch.empty_like(want)
    ops.decode_attention_fp8(q, *c.operands, *st, got, H, G, D, 40, 0.1)
    assert torch.equal(got, want)


# ---- refusals that take operands on the device ----------------------------------------------------------------------
def test_steps_without_entries():
    """A token has to belong to one."""
    H, G, D, P = 2, 1, 64, 16
    c = Cache([4], G, D, P, 66)
    q, out = rows(2, H, G, D, torch.bfloat16, 67), torch.zeros(2, H * D, dtype=torch.bfloat16, device=DEV)
    pos, seq, _ = step([(2, 2)], c.slots)
    st, k = (pos, seq, pos[:0]), torch.zeros(2, G, D, dtype=torch.bfloat16, device=DEV)
    pages, spans = torch.zeros(1, G, P, D, device=DEV), torch.tensor([[0, 0, 4, 0]], dtype=torch.int32, device=DEV)
    for call in (lambda: ops.rope_kv_write_fp8(q, *st, None, 0, *c.operands, H, G, D), lambda: ops.read_kv_fp8(*c.operands, *st, k, k),
                 lambda: ops.read_kv_fp8_spans(*c.operands, spans, P, pos[:0], pages, pages),
                 lambda: ops.decode_attention_fp8(q, *c.operands, *st, out, H, G, D, None, 1.0),
                 lambda: ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan([(2, 2)], P, DEV), *st, out, H, G, D, None, 1.0)):
        with pytest.raises(ops.KernelError, match="no entries"):
            call()


LABELS = {"k_pages": "k_pages", "v_pages": "v_pages", "k_exp": "k_exp", "v_exp": "v_exp", "block_table": "block_table|pages a request|a size", "page_size": "pages of 8"}


def on_device(x):
    if isinstance(x, torch.Tensor):
        return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=DEV).copy_(x)
    return x


def calls_on_device(cache, step, **over):
    """The calls of the host's tests with every operand on the device."""
    T, H, G, D = 3, 4, 2, 32
    qkv, out, kv = (torch.zeros(*shape, dtype=torch.bfloat16, device=DEV) for shape in ((T, (H + 2 * G) * D), (T, H * D), (T, G, D)))
    plan = ops.prefill_fp8_plan([(T, 0)], cache["page_size"], DEV)
    own = (dict(qkv=qkv), dict(k_out=kv, v_out=kv.clone()), dict(q=qkv, out=out), dict(q=qkv, out=out, plan=plan))
    calls = host._calls(*({k: on_device(v) for k, v in x.items()} for x in (cache, step)))
    return [lambda call=call, x=x: call(**{**x, **{k: on_device(v) for k, v in over.items()}}) for call, x in zip(calls, own)]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", range(len(host.BAD_CACHES)))
def test_bad_caches_on_the_device(which, bad):
    """What is refused on the host is refused by the operand's name where all of them lie on the device."""
    with pytest.raises(ops.KernelError, match=LABELS[next(iter(host.BAD_CACHES[bad]))]):
        calls_on_device(host._cache(**host.BAD_CACHES[bad]), host._step())[which]()


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", range(len(host.BAD_STEPS)))
def test_bad_steps_on_the_device(which, bad):
    name = next(iter(host.BAD_STEPS[bad]))
    with pytest.raises(ops.KernelError, match="token_seq|positions" if name == "token_seq" else name):
        calls_on_device(host._cache(), {**host._step(), **host.BAD_STEPS[bad]})[which]()


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [dict(n_heads=3), dict(n_heads=0), dict(head_dim=64), dict(n_kv_heads=4), dict(out=torch.zeros(3, 128)),
                                 dict(out=torch.zeros(3, 100, dtype=torch.bfloat16)), dict(out=torch.zeros(2, 128, dtype=torch.bfloat16)),
                                 dict(q=torch.zeros(3, 96, dtype=torch.bfloat16))])
def test_bad_attention_on_the_device(which, bad):
    with pytest.raises(ops.KernelError, match="out is a|rows of" if "out" in bad else "heads"):
        calls_on_device(host._cache(), host._step(), **bad)[which]()


@pytest.mark.parametrize("bad", [dict(n_heads=8), dict(head_dim=16), dict(inv_freq=torch.zeros(3), rotary_dim=32),
                                 dict(inv_freq=torch.zeros(16, dtype=torch.float64), rotary_dim=32),
                                 dict(inv_freq=torch.zeros(16), rotary_dim=32, cos_sin=torch.zeros(2, 16, 2))])
def test_bad_writes_on_the_device(bad):
    with pytest.raises(ops.KernelError, match="cos_sin" if "cos_sin" in bad else "inv_freq" if bad.get("inv_freq") is not None and bad["inv_freq"].dtype == torch.float64
                       else "heads"):
        calls_on_device(host._cache(), host._step(), **bad)[0]()


def test_good_calls_on_the_device():
    """The calls that the refusals above are variants of."""
    for call in calls_on_device(host._cache(), host._step()):
        call()
    torch.cuda.synchronize()


def test_a_prompt_in_a_graph():
    """A plan's lists are made before a capture; a graph made of a plan that has them follows what the buffers hold."""
    H, G, D, P = 4, 2, 64, 64
    entries = [(300, 50), (5, 20), (40, 0)]
    c = Cache([350, 25, 40], G, D, P, 68)
    q = rows(345, H, G, D, torch.bfloat16, 69)
    st, operands, plan = step(entries, c.slots), c.operands, ops.prefill_fp8_plan(entries, P, DEV)
    want, out = (torch.zeros(345, H * D, dtype=q.dtype, device=DEV) for _ in range(2))
    with pytest.raises(ops.KernelError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.prefill_attention_fp8(q, *operands, plan, *st, out, H, G, D, None, 0.1)
    ops.prefill_attention_fp8(q, *operands, plan, *st, want, H, G, D, None, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prefill_attention_fp8(q, *operands, plan, *st, out, H, G, D, None, 0.1)
    for seed in (70, 71):
        q.copy_(rows(345, H, G, D, torch.bfloat16, seed))
        graph.replay()
        ops.prefill_attention_fp8(q, *operands, plan, *st, want, H, G, D, None, 0.1)
        assert torch.equal(out, want)
    check(want, c, entries, q, H, None, 0.1, None, PROMPT_WEIGHT["bf16"])


def test_refusals_of_the_kernel_over_pages_of_128():
    H, G, D = 4, 2, 64
    q, out = torch.zeros(20, H * D, dtype=torch.bfloat16, device=DEV), torch.zeros(20, H * D, dtype=torch.bfloat16, device=DEV)
    k, table = torch.zeros(1, G, 128, D, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    items, merges, parts = ops.prefill_grouped_plan([(20, 0)], None, H, G, D)
    items = torch.from_numpy(items).to(DEV)
    good = dict(q=q, k_pages=k, v_pages=k, block_table=table, items=items, out=out, n_heads=H, n_kv_heads=G, head_dim=D, window=None, scale=1.0)
    ops.prefill_attention_grouped(**good)
    for bad in (dict(q=q.float()), dict(q=q.float(), out=out.float(), k_pages=k.float(), v_pages=k.float()), dict(v_pages=k[:0]), dict(k_pages=k[:, :1]),
                dict(k_pages=k[:, :, :64], v_pages=k[:, :, :64]), dict(block_table=table.long()), dict(items=items.long()), dict(items=items[:, :7]),
                dict(out=out[:, :64]), dict(n_heads=8), dict(n_heads=3), dict(n_kv_heads=4), dict(scale=0.0), dict(scale=-1.0), dict(parts=3),
                dict(parts=1, merges=torch.zeros(1, 3, dtype=torch.int32, device=DEV))):
        with pytest.raises(ops.KernelError):
            ops.prefill_attention_grouped(**{**good, **bad})


def test_pairs_of_cosine_and_sine_off_their_grid():
    H, G, D, P = 2, 1, 64, 16
    c = Cache([4], G, D, P, 81)
    q, cs = rows(2, H, G, D, torch.bfloat16, 82), torch.zeros(2 * 32 * 2 + 1, device=DEV)
    with pytest.raises(ops.KernelError):
        ops.rope_kv_write_fp8(q, *step([(2, 2)], c.slots), torch.ones(32, device=DEV), 64, *c.operands, H, G, D, cos_sin=cs[1:].reshape(2, 32, 2))


def test_a_plan_of_another_device():
    H, G, D, P = 2, 1, 64, 16
    c = Cache([20], G, D, P, 72)
    q, out = rows(20, H, G, D, torch.bfloat16, 73), torch.zeros(20, H * D, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ops.KernelError, match="a plan made for cpu"):
        ops.prefill_attention_fp8(q, *c.operands, ops.prefill_fp8_plan([(20, 0)], P, "cpu"), *step([(20, 0)], c.slots), out, H, G, D, None, 1.0)
