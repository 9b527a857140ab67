"""The 8-bit cache on the CPU: the form's definition, what the entry points refuse, how a prompt step is planned."""
import math

import pytest
import torch

import plain_fp8_cache as plain
from ferrox_b200.cache.specs import CacheSpec, KvCacheSpec, PagedSpec, PagedTensorSpec, in_8_bits
from ferrox_b200.config.registry import resolve
from ferrox_b200.kernels import ops
from ferrox_b200.parts.build import build_model
from tiny_configs import TINY_A


# ---- the definition -------------------------------------------------------------------------------------------------
def test_the_plain_form_rounds_to_nearest_even():
    v, e = plain.quantise(torch.tensor([[448.0, 17.0, 19.0, 18.0, 0.0, -17.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10]]))
    assert e.tolist() == [127]
    assert v.tolist() == [[448.0, 16.0, 20.0, 18.0, 0.0, -16.0, 2.0 ** -9, 0.0, 2 * 2.0 ** -9]]


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.5, 1), (449.0, 1), (224.0, -1), (3.3e38, 120), (1e-40, -119), (0.0, -119)])
def test_the_exponent_is_the_smallest_that_fits(amax, e):
    v, got = plain.quantise(torch.tensor([[amax, 0.0]], dtype=torch.float64))
    assert int(got[0]) == e + 127 and float(v.abs().max()) <= 448.0


def test_an_error_is_at_most_half_a_step():
    x = torch.randn(50, 64, dtype=torch.float64) * torch.exp(torch.randn(50, 1, dtype=torch.float64) * 5)
    y = plain.values(*plain.quantise(x))
    small = torch.exp2(plain.quantise(x)[1].double() - 127)[:, None] * 2.0 ** -10      # half a step of the smallest numbers
    assert ((x - y).abs() <= torch.maximum(x.abs() * 2.0 ** -4, small)).all()


def test_values_are_exact_in_16_bits():
    exps = torch.arange(8, 248)
    x = plain.values(plain.TABLE[:127][None].expand(240, -1), exps)
    x = x[x <= plain.MOST]
    assert torch.equal(x.to(torch.bfloat16).double(), x)


# ---- specs and models -----------------------------------------------------------------------------------------------
def test_pages_in_8_bits():
    p = in_8_bits(KvCacheSpec(3, 48, window=7))
    assert [(t.name, t.dtype, t.page_shape(16)) for t in p.tensors] == [
        ("k", torch.float8_e4m3fn, (3, 16, 48)), ("v", torch.float8_e4m3fn, (3, 16, 48)), ("k_exp", torch.uint8, (3, 16)),
        ("v_exp", torch.uint8, (3, 16))] and p.window == 7
    with pytest.raises(ValueError, match="8-bit cache"):
        in_8_bits(PagedSpec((PagedTensorSpec("kv", (64,)),)))


def test_a_model_gives_its_caches_in_8_bits():
    model = build_model(resolve(TINY_A)[1])
    assert all(isinstance(c, CacheSpec) and len(c.paged.tensors) == 4 for c in model.cache_specs("fp8"))
    assert all(len(c.paged.tensors) == 2 for c in model.cache_specs())
    with pytest.raises(ValueError, match="kv_cache='int4'"):
        model.cache_specs("int4")


def test_a_layer_that_cannot_is_refused_by_name():
    from zanezen_configs import ZANEZEN_A
    model = build_model(resolve(ZANEZEN_A)[1])
    with pytest.raises(ValueError, match="not held in 8 bits"):
        model.cache_specs("fp8")


# ---- refusals: before anything is launched --------------------------------------------------------------------------
def _cache(pages=3, G=2, P=16, D=32, **other):
    c = dict(k_pages=torch.zeros(pages, G, P, D, dtype=torch.float8_e4m3fn), v_pages=torch.zeros(pages, G, P, D, dtype=torch.float8_e4m3fn),
             k_exp=torch.zeros(pages, G, P, dtype=torch.uint8), v_exp=torch.zeros(pages, G, P, dtype=torch.uint8),
             block_table=torch.zeros(2, 4, dtype=torch.int32), page_size=P)
    c.update(other)
    return c


def _step(T=3):
    return dict(positions=torch.arange(T, dtype=torch.int32), token_seq=torch.zeros(T, dtype=torch.int32), seq_slot=torch.zeros(1, dtype=torch.int32))


BAD_CACHES = [
    dict(k_pages=torch.zeros(3, 2, 16, 32)), dict(v_pages=torch.zeros(3, 2, 16, 32, dtype=torch.float8_e5m2)),
    dict(k_exp=torch.zeros(3, 2, 16)), dict(v_exp=torch.zeros(3, 2, 15, dtype=torch.uint8)), dict(page_size=8),
    dict(v_pages=torch.zeros(3, 2, 16, 64, dtype=torch.float8_e4m3fn)), dict(block_table=torch.zeros(2, 4, dtype=torch.int64)),
    dict(block_table=torch.zeros(8, dtype=torch.int32)), dict(block_table=torch.zeros(4, 2, dtype=torch.int32).T),
    dict(k_pages=torch.zeros(3, 16, 2, 32, dtype=torch.float8_e4m3fn).transpose(1, 2)), dict(block_table=torch.zeros(2, 0, dtype=torch.int32)),
]
BAD_STEPS = [dict(positions=torch.zeros(3, dtype=torch.int64)), dict(token_seq=torch.zeros(2, dtype=torch.int32)),
             dict(seq_slot=torch.zeros(1, dtype=torch.int64)), dict(positions=torch.zeros(6, dtype=torch.int32)[::2])]


def _calls(cache, step, T=3, H=4, G=2, D=32, dtype=torch.bfloat16, **over):
    qkv, out = torch.zeros(T, (H + 2 * G) * D, dtype=dtype), torch.zeros(T, H * D, dtype=dtype)
    rows = torch.zeros(T, G, D, dtype=dtype)
    plan = ops.prefill_fp8_plan([(T, 0)], cache["page_size"], "cpu")
    shape = dict(n_heads=H, n_kv_heads=G, head_dim=D)
    attend = dict(window=None, scale=1.0)
    return [
        lambda **o: ops.rope_kv_write_fp8(**{**dict(qkv=qkv, inv_freq=None, rotary_dim=0), **cache, **step, **shape, **over, **o}),
        lambda **o: ops.read_kv_fp8(**{**cache, **step, **dict(k_out=rows, v_out=rows), **over, **o}),
        lambda **o: ops.decode_attention_fp8(**{**dict(q=qkv, out=out), **cache, **step, **shape, **attend, **over, **o}),
        lambda **o: ops.prefill_attention_fp8(**{**dict(q=qkv, out=out, plan=plan), **cache, **step, **shape, **attend, **over, **o}),
    ]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", range(len(BAD_CACHES)))
def test_bad_caches(which, bad):
    with pytest.raises(ops.KernelError):
        _calls(_cache(**BAD_CACHES[bad]), _step())[which]()


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("bad", range(len(BAD_STEPS)))
def test_bad_steps(which, bad):
    with pytest.raises(ops.KernelError):
        _calls(_cache(), {**_step(), **BAD_STEPS[bad]})[which]()


@pytest.mark.parametrize("which", range(4))
def test_tensors_of_the_host(which):
    with pytest.raises(ops.KernelError, match="an operand on cpu"):
        _calls(_cache(), _step())[which]()


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [dict(n_heads=3), dict(n_heads=0), dict(head_dim=64), dict(n_kv_heads=4), dict(window=0), dict(window=-3),
                                 dict(softcap=0.0), dict(softcap=-1.0), dict(scale=math.inf), dict(scale=math.nan),
                                 dict(out=torch.zeros(3, 128)), dict(out=torch.zeros(3, 100, dtype=torch.bfloat16)),
                                 dict(out=torch.zeros(2, 128, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 96, dtype=torch.bfloat16))])
def test_bad_attention(which, bad):
    with pytest.raises(ops.KernelError, match="fp8"):
        _calls(_cache(), _step())[which](**bad)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("bad", [dict(softcap=math.inf), dict(softcap=math.nan), dict(softcap=1e39), dict(softcap=3e38), dict(softcap=1e-46), dict(scale=1e39),
                                 dict(scale=-3e38), dict(softcap=1e-30, scale=1e10), dict(softcap=1e-44), dict(softcap=10 ** 400), dict(window=1 << 31)])
def test_scores_beyond_32_bits(which, bad):
    """A cap of which 32 bits hold 0 would be none at all, an infinite one or an infinite scale no number: refused, whatever the operands."""
    with pytest.raises(ops.KernelError, match="softcap="):
        _calls(_cache(), _step())[which](**bad)
    if which == 3:
        with pytest.raises(ops.KernelError, match="prefill_attention_grouped: window=.* softcap="):
            ops.prefill_attention_grouped(*[torch.zeros(1)] * 6, 4, 2, 32, **{**dict(window=None, scale=1.0), **bad})


@pytest.mark.parametrize("which", [2, 3])
def test_scales_so_far_over_their_cap_that_nothing_times_them_is_no_number(which):
    """2^127 times 2 log2(e), which the prompt kernel multiplies a score with, is infinite, and a score may be 0."""
    for over, refused in ((2.0 ** 126, True), (2.0 ** 125, False)):
        with pytest.raises(ops.KernelError, match="2\\^125 times the cap" if refused else "an operand on cpu"):
            _calls(_cache(), _step())[which](softcap=0.5, scale=over / 2)


@pytest.mark.parametrize("which", [2, 3])
@pytest.mark.parametrize("good", [dict(softcap=1e30), dict(softcap=1e-30), dict(scale=1e37, softcap=1.0), dict(scale=-1e-50), dict(scale=0.0, softcap=2.0 ** -149),
                                  dict(window=(1 << 31) - 1)])
def test_scores_within_32_bits(which, good):
    with pytest.raises(ops.KernelError, match="an operand on cpu"):
        _calls(_cache(), _step())[which](**good)


@pytest.mark.parametrize("bad", [dict(n_heads=8), dict(head_dim=16), dict(inv_freq=torch.zeros(3), rotary_dim=32),
                                 dict(inv_freq=torch.zeros(16, dtype=torch.float64), rotary_dim=32),
                                 dict(inv_freq=torch.zeros(16), rotary_dim=32, cos_sin=torch.zeros(2, 16, 2))])
def test_bad_writes(bad):
    with pytest.raises(ops.KernelError, match="rope_kv_write_fp8"):
        _calls(_cache(), _step())[0](**bad)


def test_bad_reads():
    c, slot = _cache(), torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(2, 2, 16, 32)
    for spans, rows, a, b in [(torch.zeros(1, 4, dtype=torch.int32), 30, k, k), (torch.zeros(4, dtype=torch.int32), 32, k, k),
                              (torch.zeros(0, 4, dtype=torch.int32), 32, k, k), (torch.zeros(1, 4, dtype=torch.int64), 32, k, k),
                              (torch.zeros(1, 4, dtype=torch.int32), 32, k, k.bfloat16()), (torch.zeros(1, 4, dtype=torch.int32), 48, k, k)]:
        with pytest.raises(ops.KernelError, match="read_kv_fp8"):
            ops.read_kv_fp8_spans(**c, spans=spans, n_rows=rows, seq_slot=slot, k_out=a, v_out=b)


def test_a_plan_of_another_step():
    c, s = _cache(), _step()
    for plan in (ops.prefill_fp8_plan([(2, 0)], 16, "cpu"), ops.prefill_fp8_plan([(3, 0)], 32, "cpu"), ops.prefill_fp8_plan([(2, 0), (1, 5)], 16, "cpu")):
        with pytest.raises(ops.KernelError):
            _calls(c, s)[3](plan=plan)
    for entries, page in (([(-1, 0)], 16), ([(1, -1)], 16), ([(1, 0)], 0)):
        with pytest.raises(ops.KernelError, match="prefill_fp8_plan"):
            ops.prefill_fp8_plan(entries, page, "cpu")


def test_every_error_of_the_library_has_its_words():
    import os
    import re
    from ferrox_b200.kernels import lib
    codes = set()
    for name in ("common.cuh", "no_alloc.h"):
        with open(os.path.join(lib.CSRC, name)) as f:
            codes |= {int(c) for c in re.findall(r"#define FX_ERR_\w+ (-\d+)", f.read())}
    assert codes == set(ops._ERRORS) and len(set(ops._ERRORS.values())) == len(codes) >= 6


def test_no_kv_heads():
    """Nothing to write for, and nothing for a query to read: refused where the heads are named (the queries would stay unrotated)."""
    with pytest.raises(ops.KernelError, match="pages of 16 positions"):
        ops._check_fp8("x", (3, 0, 16, 32), 16, 0, 32)
    ops._check_fp8("x", (3, 0, 16, 32), 16, None, None)                     # (reading none of them back is nothing to do)
    ops._check_fp8("x", (3, 2, 16, 32), 16, 2, 32)


# ---- how a prompt step is planned -----------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [None, 5, 40])
@pytest.mark.parametrize("most", [1, 3000, 1 << 30])
def test_parts_hold_what_the_tokens_see(window, most, monkeypatch):
    monkeypatch.setattr(ops, "FP8_READ_BACK_MAX", most)
    P, entries = ops.FP8_READ_PAGE, [(40, 0), (3, 100), (17, 33), (9, 0), (0, 12), (200, 7), (8, 0)]
    plan = ops.prefill_fp8_plan(entries, 16, "cpu")
    few = plan.few(window, 10).tolist()
    placed = len(few)
    seen, first = set(few), [0]
    for n, _ in entries:
        first.append(first[-1] + n)
    for tok0, n, own, spans, rows, table, slots in plan.parts(window, 10):
        assert sum(m for m, _ in own) == n and slots.tolist() == list(range(len(own))) and (len(own) == 1 or rows * 10 <= most)
        at, row = tok0, 0
        for (m, start), (b, seen_from, end, r), pages in zip(own, spans.tolist(), table.tolist()):
            p0 = seen_from // P * P
            assert (m, start) == entries[b] and at == first[b] and end == start + m and r == row + seen_from - p0
            assert seen_from == ops.first_key(start, window)
            for p in range(len(pages)):
                inside = p0 <= p * P < end
                assert pages[p] == (row // P + p - p0 // P if inside else -1)
            seen |= set(range(at, at + m))
            at += m
            placed += m
            row += -(-(end - p0) // P) * P
        assert row == rows
    assert seen == set(range(first[-1])) and placed == first[-1] and len(few) == 8 + (3 if most < 1 << 30 else 0)      # (the 3 go with their neighbours)


@pytest.mark.parametrize("keys,parts", [(0, 2), (102, 2), (103, 1)])
def test_few_tokens_between_others(keys, parts, monkeypatch):
    monkeypatch.setattr(ops, "FP8_JOIN_KEYS", keys)
    plan = ops.prefill_fp8_plan([(2, 5), (40, 0), (3, 100), (0, 4), (17, 33), (5, 0)], 16, "cpu")
    found = plan.parts(None, 10)
    assert len(found) == parts and found[0][0] == 2
    few = list(range(2)) + list(range(62, 67))
    assert plan.few(None, 10).tolist() == (few if parts == 1 else few[:2] + [42, 43, 44] + few[2:])
    assert plan.few(8, 10).tolist() != [] and len(plan.parts(8, 10)) == (2 if keys < 11 else 1)      # (the 3 see 10 keys there)


@pytest.mark.parametrize("kind,heads,kv_heads,dim", [("grouped", 28, 4, 128), ("capped", 28, 4, 128), ("tc", 16, 16, 128), ("mma", 16, 4, 256), ("f32", 16, 4, 128)])
def test_what_goes_token_by_token(kind, heads, kv_heads, dim):
    def choice(entries, window=None):
        return ops.fp8_token_by_token(kind, entries, window, heads, kv_heads, dim, sms=148)
    assert choice([(1, 5000)] * 30) and choice([(8, 0), (3, 100)]) and choice([])
    assert choice([(12, 100)]) and choice([(1, 4000)] * 40 + [(12, 20)])
    assert not choice([(2048, 0)]) and not choice([(300, 3700)] * 6)
    sizes = [choice([(n, 1000)] * 4) for n in (9, 16, 32, 64, 128, 256, 1024)]
    assert sizes == sorted(sizes, reverse=True)                             # (once tiled, tiled with more tokens)


# ---- one plan, layers of several shapes -----------------------------------------------------------------------------
def _prompt_layer(plan, monkeypatch, heads, kv_heads, dim, dtype=torch.bfloat16, window=None, dim_out=0):
    """What a layer of a prompt step hands to the kernels over read-back pages: [(first token, tokens, block table, tile lists)], the
    launches put aside."""
    T, found = plan.n_tokens, []

    def look(name, q, *rest):
        x = ops.BF16 if q.dtype == torch.bfloat16 else ops.F32
        return (None, 0, x, *[256] * 12, 9, kv_heads, plan.page_size, dim, 1, 9, T, len(plan.entries), heads * dim, heads * dim, 1, -1, q.stride(0), heads * dim + dim_out)

    def kernel(rows, stays):
        def record(q, k, v, table, *lists_and_rest, **kw):
            at = (q.data_ptr() - q_all.data_ptr()) // (q_all.stride(0) * q_all.element_size())
            found.append((at, q.shape[0], table, rows([x for x in lists_and_rest if isinstance(x, torch.Tensor) and x.dim() == 2 and x.dtype == torch.int32])))
            return stays
        return record

    q_all = torch.zeros(T, heads * dim, dtype=dtype)
    monkeypatch.setattr(ops, "_look_at_attention_fp8", look)
    monkeypatch.setattr(ops, "sm_count", lambda: 148)
    monkeypatch.setattr(ops, "fp8_token_by_token", lambda *a: False)
    monkeypatch.setattr(ops, "read_kv_fp8_spans", lambda *a, **k: None)
    monkeypatch.setattr(ops, "decode_attention_fp8", lambda *a, **k: None)
    monkeypatch.setattr(ops, "prefill_attention_grouped", kernel(lambda t: t[0][:, :3], None))
    monkeypatch.setattr(ops, "prefill_attention_tc", kernel(lambda t: t[0][:, :3], None))
    monkeypatch.setattr(ops, "prefill_attention", kernel(lambda t: t[0][:, :3], None))
    monkeypatch.setattr(ops, "prefill_attention_f32_tc", kernel(lambda t: t[0][:, :3], None))
    monkeypatch.setattr(ops, "prefill_attention_f32", kernel(lambda t: t[0][:, :3], None))
    ops.prefill_attention_fp8(q_all, *[None] * 5, plan.page_size, plan, None, None, None, torch.zeros(T, heads * dim, dtype=dtype), heads, kv_heads, dim,
                              window, 1.0)
    return found


SHAPES = [("grouped", dict(heads=16, kv_heads=16, dim=64)), ("grouped", dict(heads=16, kv_heads=16, dim=128)), ("grouped", dict(heads=16, kv_heads=4, dim=64)),
          ("tc", dict(heads=130, kv_heads=1, dim=64)), ("tc", dict(heads=130, kv_heads=1, dim=128)),
          ("mma", dict(heads=130, kv_heads=1, dim=144)), ("mma", dict(heads=130, kv_heads=1, dim=256)),
          ("f32", dict(heads=16, kv_heads=16, dim=64, dtype=torch.float32)), ("f32", dict(heads=16, kv_heads=4, dim=64, dtype=torch.float32)),
          ("f32", dict(heads=16, kv_heads=4, dim=68, dtype=torch.float32)), ("f32", dict(heads=16, kv_heads=2, dim=68, dtype=torch.float32))]


@pytest.mark.parametrize("a", range(len(SHAPES)))
@pytest.mark.parametrize("b", range(len(SHAPES)))
def test_a_plan_serves_layers_that_are_cut_differently(a, b, monkeypatch):
    """A step is cut into portions by the bytes that a layer reads back, so that layers of other heads, head sizes or types have other
    portions.  Every list names entries of its own portion only and holds all of its tokens, whatever layer has used the plan before."""
    monkeypatch.setattr(ops, "FP8_READ_BACK_MAX", 4 * 512 * 2 * 16 * 64 * 2)              # (four entries of the first shape)
    plan = ops.prefill_fp8_plan([(40, 460)] * 6, 64, "cpu")
    for kind, shape in (SHAPES[a], SHAPES[b]):
        row_bytes = 2 * shape["kv_heads"] * shape["dim"] * (4 if shape.get("dtype") else 2)
        found = _prompt_layer(plan, monkeypatch, **shape)
        assert sum(n for _, n, _, _ in found) == 240
        assert all(n <= 40 or n // 40 * 512 * row_bytes <= ops.FP8_READ_BACK_MAX for _, n, _, _ in found)
        at = 0
        for first, n, table, tiles in found:
            assert first == at and table.shape[0] == n // 40
            covered = sorted((t, t + m, e) for t, m, e in set(map(tuple, tiles.tolist())))
            assert covered[0][0] == 0 and covered[-1][1] == n and all(x[1] == y[0] for x, y in zip(covered, covered[1:]))
            assert all(0 <= e < table.shape[0] and t // 40 == e == (end - 1) // 40 for t, end, e in covered)
            at += n


# ---- a plan on several streams --------------------------------------------------------------------------------------
def test_a_capture_does_not_stand_for_the_stream_before_it(monkeypatch):
    """The stream that copied a plan's lists is waited for by the next one that is no capture's, a capture between them or not."""
    waited, capturing = [], False

    class Stream:
        def wait_stream(self, other):
            waited.append(other)

    monkeypatch.setattr(ops, "_stream_of", lambda pointer, device: pointer)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    plan = ops.prefill_fp8_plan([(20, 0)], 16, "cpu")
    plan.on_stream(1)
    plan.on_stream(1)
    assert waited == []
    capturing = True
    plan.on_stream(2)
    assert waited == []
    capturing = False
    plan.on_stream(3)
    assert waited == [1]
    plan.on_stream(1)
    plan.on_stream(3)
    assert waited == [1, 3, 1]
