"""An 8-bit key-value cache: keys and values quantised as they are written into pages, read back, and read by attention.

A position of one kv head stores ``head_dim`` bytes of e4m3 (four exponent bits, three mantissa bits) and one byte E, the
exponent of a power of two: element i stands for e4m3(byte i) * 2^(E - 127).  Keys and values lie in pages
[pages, kv heads, page, head_dim] with their exponents in [pages, kv heads, page]; a block table names the pages of a
request in order.  With a = the largest |x| of the row, e is the smallest whole number with a <= 448 * 2^e (448: the
largest e4m3 value), at least -119, E = e + 127, and byte i is x_i / 2^e rounded to nearest, ties to even.  Both steps are
exact but for that one rounding, so what is written is the same whatever computes it.

Four operators:

* ``write``:  the k and v rows of a step's fused [q | k | v] rows into the pages, and the step's positions read back
* ``read``:   the positions of whole requests back into pages of 16 or 32 bits (zeros behind a request's last position)
* ``decode``: attention of one new token a request over its pages: out = softmax(cap(scale q . k)) v over the positions
  max(0, p - window + 1) .. p, cap(s) = c tanh(s / c); query head h reads kv head h / (heads / kv heads)
* ``prompt``: the same for portions of several tokens a request, behind what the request's pages hold already
"""
from __future__ import annotations

import math

import torch

own = False

PAGE_SLACK = 2                 # columns of a block table behind the longest request's
LONGEST, SHORTEST = 448.0, -119


# ---- cases ----------------------------------------------------------------------------------------------------------
def _case(name, op, dtype, requests, longest, new, heads, kv_heads, dim, page=64, window=0, softcap=0.0):
    return dict(name=name, op=op, dtype=dtype, requests=requests, longest=longest, new=new, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, window=window, softcap=softcap)


def listed():
    return [
        # a decode step of a serving engine: one token a request
        _case("write 32 tokens", "write", "bf16", 32, 2048, 1, 28, 4, 128),
        # a prompt step: portions of unequal lengths, together some 2,000 tokens
        _case("write prompt portions", "write", "bf16", 4, 1024, 1024, 16, 16, 128),
        # one request's context for a 32-bit model with short heads, odd lengths and small pages
        _case("read 517 positions f32", "read", "f32", 1, 517, 1, 4, 2, 64, page=16),
        # a few long contexts, handed to a kernel that takes 16-bit pages
        _case("read long contexts", "read", "bf16", 4, 32768, 1, 28, 4, 128),
        # the smallest step there is: one request that has just begun
        _case("decode 1 x 37", "decode", "bf16", 1, 37, 1, 16, 16, 128),
        # a full serving batch
        _case("decode 64 x 4096", "decode", "bf16", 64, 4096, 1, 28, 4, 128),
        # one very long conversation, alone on the machine
        _case("decode 1 x 131072", "decode", "bf16", 1, 131072, 1, 28, 4, 128),
        # a layer with a window and capped scores, one kv head a query head
        _case("decode window capped", "decode", "bf16", 24, 4000, 1, 16, 16, 128, window=1024, softcap=30.0),
        # a 32-bit model
        _case("decode f32", "decode", "f32", 8, 2000, 1, 16, 4, 128),
        # a prompt of 2,048 tokens
        _case("prompt 2048", "prompt", "bf16", 1, 2048, 2048, 16, 16, 128),
        # portions behind what is cached already: turns of conversations
        _case("prompt turns", "prompt", "bf16", 6, 4096, 300, 28, 4, 128),
        # short prompts of a 32-bit model
        _case("prompt f32", "prompt", "f32", 3, 300, 300, 4, 2, 64),
    ]


def _pick(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most = {k: max(most.get(k, 0.0), w[k]) for k in w}
    while True:
        op = rng.choice(["write", "read", "decode", "decode", "prompt"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        heads, kv_heads = rng.choice([(16, 16), (28, 4), (16, 4), (4, 2), (6, 3), (32, 2), (8, 1), (5, 5)])
        dim = rng.choice([64, 128, 128, 128, 48, 96, 80, 256])
        page = rng.choice([16, 32, 64, 64, 64, 128])
        requests = _pick(rng, 1, 64)
        longest = _pick(rng, 1, 65536 if op in ("decode", "read") else 4096)
        new = 1 if op in ("decode", "read") else _pick(rng, 1, min(longest, 2048))
        window = _pick(rng, 1, 2 * longest) if op in ("decode", "prompt") and rng.random() < 0.3 else 0
        softcap = rng.choice([15.0, 30.0, 50.0]) if op in ("decode", "prompt") and rng.random() < 0.25 else 0.0
        c = _case("", op, dtype, requests, longest, new, heads, kv_heads, dim, page, window, softcap)
        del c["name"]
        w = work(c)
        scores = requests * heads * new * longest                       # (the plain form holds them all)
        gathered = requests * longest * kv_heads * dim
        if all(w[k] <= most[k] for k in w) and scores <= 2.5e8 and gathered <= 2 ** 27 and (dtype == "bf16" or scores * dim < 2e10):
            return c


def _lengths(case):
    """[(positions that the request holds with this step's, new ones)], the same for every seed: from the longest down to
    a third of it, the last request of several the shortest there is."""
    n, longest, new = case["requests"], case["longest"], case["new"]
    out = []
    for b in range(n):
        share = 1.0 if n == 1 else 1.0 - (2.0 / 3.0) * b / (n - 1)
        length = max(1, int(longest * share) - (b * 7) % 11)
        if n > 2 and b == n - 1:
            length = min(length, new)
        fresh = max(1, min(length, new - (b * 13) % max(1, new // 3 + 1)))
        out.append((length, fresh))
    return out


def _keys_seen(case):
    """(query, key) pairs, and distinct positions read."""
    window, pairs, positions = case["window"], 0, 0
    for length, fresh in _lengths(case):
        first = length - fresh
        reach = window if window else length
        for_all = fresh * first + fresh * (fresh + 1) // 2
        if window:
            full = max(0, length - max(first, window - 1))              # queries whose window is full
            part = fresh - full
            for_all = full * window + part * first + part * (part + 1) // 2
        pairs += for_all
        positions += min(length, reach + fresh - 1)
    return pairs, positions


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    kvh, h, d = case["kv_heads"], case["heads"], case["dim"]
    tokens = sum(f for _, f in _lengths(case))
    held = sum(n for n, _ in _lengths(case))
    row = 2 * kvh * (d + 1)                                             # a position's bytes in the pages
    if case["op"] == "write":
        return {"bytes": float(tokens * (2 * kvh * d * es * 2 + 2 * row)), "flops": float(tokens * 2 * kvh * d * 2)}
    if case["op"] == "read":
        rows = sum(-(-n // case["page"]) * case["page"] for n, _ in _lengths(case))
        return {"bytes": float(held * row + rows * 2 * kvh * d * es), "flops": float(held * 2 * kvh * d)}
    pairs, positions = _keys_seen(case)
    return {"bytes": float(positions * row + tokens * 2 * h * d * es), "flops": float(pairs * h * d * 4)}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _power(e):
    """2^e in 32 bits, made of its bits; e = -127: 0."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """(bytes of e4m3, exponent bytes) of rows x [..., dim] in 32 bits."""
    a = x.abs().amax(-1)
    m, e = torch.frexp(a)                                               # a = m 2^e, m in [1/2, 1)
    e = torch.where(m <= 0.875, e - 9, e - 8)                           # 448 = 0.875 * 2^9
    e = torch.where(a > 0, e, torch.full_like(e, SHORTEST)).clamp_min(SHORTEST)
    q = (x * _power(-e)[..., None]).to(torch.float8_e4m3fn)
    return q.view(torch.uint8), (e + 127).to(torch.uint8)


def _values(q, exps):
    """What bytes and exponents stand for, in 32 bits."""
    return q.view(torch.float8_e4m3fn).float() * _power(exps.to(torch.int32) - 127)[..., None]


def prepare(case, seed):
    """The step's rows and its index arrays as an engine has them, pages filled with earlier steps' keys and values, the
    outputs' buffers.  Rows have the spread of projected activations: channels of unequal size, a few large ones."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, dt = "cuda", _dtype(case)
    kvh, h, d, page = case["kv_heads"], case["heads"], case["dim"], case["page"]
    lens = _lengths(case)
    n = len(lens)
    width = -(-max(x for x, _ in lens) // page) + PAGE_SLACK
    need = [-(-x // page) for x, _ in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu()
    slots = torch.randperm(n + 3, generator=g, device=dev)[:n].to(torch.int32).cpu()
    table = torch.full((n + 3, width), -1, dtype=torch.int32)
    at = 0
    for b in range(n):
        table[slots[b], :need[b]] = order[at:at + need[b]]
        at += need[b]
    channel = torch.exp(0.5 * torch.randn(kvh, 1, d, generator=g, device=dev))
    channel = torch.where(torch.rand(kvh, 1, d, generator=g, device=dev) < 0.03, channel * 6.0, channel)

    def rows(factor):
        q = torch.empty(pages, kvh, page, d, dtype=torch.uint8, device=dev)
        e = torch.empty(pages, kvh, page, dtype=torch.uint8, device=dev)
        for i in range(0, pages, 512):                                  # (in parts: 32-bit rows of all pages at once are large)
            x = torch.randn(min(512, pages - i), kvh, page, d, generator=g, device=dev) * factor
            q[i:i + 512], e[i:i + 512] = _quantised(x)
        return q.view(torch.float8_e4m3fn), e

    k_pages, k_exp = rows(channel)
    v_pages, v_exp = rows(0.7)
    positions = torch.cat([torch.arange(x - f, x) for x, f in lens]).to(torch.int32)
    token_seq = torch.cat([torch.full((f,), b) for b, (_, f) in enumerate(lens)]).to(torch.int32)
    t = positions.numel()
    qkv = torch.randn(t, (h + 2 * kvh) * d, generator=g, device=dev)
    qkv[:, h * d:(h + kvh) * d] *= channel.reshape(1, -1)
    s = dict(case=case, lens=lens, k_pages=k_pages, k_exp=k_exp, v_pages=v_pages, v_exp=v_exp, table=table.to(dev),
             slots=slots.to(dev), positions=positions.to(dev), token_seq=token_seq.to(dev), qkv=qkv.to(dt),
             scale=1.0 / math.sqrt(d), window=case["window"] or None, softcap=case["softcap"] or None)
    if case["op"] == "write":
        s["k"], s["v"] = (torch.zeros(t, kvh, d, dtype=dt, device=dev) for _ in range(2))
    elif case["op"] == "read":
        first = [0]
        for x in need:
            first.append(first[-1] + x * page)
        # (request, first position, end, first row), an engine's list of what a step needs read back
        s["spans"] = torch.tensor([[b, 0, x, first[b]] for b, (x, _) in enumerate(lens)], dtype=torch.int32, device=dev)
        s["rows"] = first[-1]
        s["k"], s["v"] = (torch.zeros(first[-1] // page, kvh, page, d, dtype=dt, device=dev) for _ in range(2))
    else:
        s["out"] = torch.zeros(t, h * d, dtype=dt, device=dev)
        s["new"] = max(f for _, f in lens)
    if own and case["op"] == "prompt":
        from ferrox_b200.kernels import ops
        # the host's list of a step's tiles: an engine makes it once a step for all its layers
        s["plan"] = ops.prefill_fp8_plan([(f, x - f) for x, f in lens], page, dev)
    return s


# ---- the operators --------------------------------------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from ferrox_b200.kernels import ops

    c = s["case"]
    kvh, h, d, page = c["kv_heads"], c["heads"], c["dim"], c["page"]
    cache = (s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"], s["table"], page)
    step = (s["positions"], s["token_seq"], s["slots"])
    if c["op"] == "write":
        ops.rope_kv_write_fp8(s["qkv"], *step, None, 0, *cache, h, kvh, d)
        ops.read_kv_fp8(*cache, *step, s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    if c["op"] == "read":
        ops.read_kv_fp8_spans(*cache, s["spans"], s["rows"], s["slots"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    if c["op"] == "decode":
        return ops.decode_attention_fp8(s["qkv"], *cache, *step, s["out"], h, kvh, d, s["window"], s["scale"], softcap=s["softcap"])
    return ops.prefill_attention_fp8(s["qkv"], *cache, s["plan"], *step, s["out"], h, kvh, d, s["window"], s["scale"],
                                     softcap=s["softcap"])


def _places(s, positions, request):
    """(page, place in it) of positions [...] of requests [...]; the first page where there is none."""
    page = s["case"]["page"]
    p = s["table"][s["slots"][request].long(), (positions // page).long()].long()
    return p.clamp_min(0), (positions % page).long()


def _gathered(s, length):
    """Keys and values of all requests' first ``length`` positions, [requests, kv heads, length, dim] in 32 bits."""
    n = len(s["lens"])
    pos = torch.arange(length, device="cuda")[None, :].expand(n, -1)
    limit = s["table"].shape[1] * s["case"]["page"]
    at, i = _places(s, pos.clamp_max(limit - 1), torch.arange(n, device="cuda")[:, None].expand(-1, length))
    return tuple(_values(q.view(torch.uint8)[at, :, i], e[at, :, i]).transpose(1, 2) for q, e in
                 ((s["k_pages"], s["k_exp"]), (s["v_pages"], s["v_exp"])))


def _run_plain(s):
    c = s["case"]
    kvh, h, d, page, dt = c["kv_heads"], c["heads"], c["dim"], c["page"], _dtype(s["case"])
    if c["op"] == "write":
        at, i = _places(s, s["positions"], s["token_seq"].long())
        k, v = s["qkv"][:, h * d:].float().reshape(-1, 2, kvh, d).unbind(1)
        kq, ke = _quantised(k)
        vq, ve = _quantised(v)
        s["k_pages"].view(torch.uint8)[at, :, i] = kq
        s["v_pages"].view(torch.uint8)[at, :, i] = vq
        s["k_exp"][at, :, i] = ke
        s["v_exp"][at, :, i] = ve
        return {"k": _values(s["k_pages"].view(torch.uint8)[at, :, i], s["k_exp"][at, :, i]).to(dt),
                "v": _values(s["v_pages"].view(torch.uint8)[at, :, i], s["v_exp"][at, :, i]).to(dt)}
    lens = torch.tensor([x for x, _ in s["lens"]], device="cuda")
    if c["op"] == "read":
        row = torch.arange(s["rows"], device="cuda")
        b = torch.searchsorted(s["spans"][:, 3].contiguous(), row, right=True) - 1
        pos = row - s["spans"][b, 3]
        at, i = _places(s, pos, b)
        there = (pos < lens[b])[:, None, None]
        out = [torch.where(there, _values(q.view(torch.uint8)[at, :, i], e[at, :, i]), 0.0).to(dt)
               for q, e in ((s["k_pages"], s["k_exp"]), (s["v_pages"], s["v_exp"]))]
        k, v = (x.reshape(-1, page, kvh, d).transpose(1, 2).contiguous() for x in out)
        return {"k": k, "v": v}
    # decode and prompt: every request's queries padded to the longest portion, its keys to the longest request
    n, longest, new = len(s["lens"]), max(x for x, _ in s["lens"]), s["new"]
    k, v = _gathered(s, longest)
    fresh = torch.tensor([f for _, f in s["lens"]], device="cuda")
    first_row = torch.cumsum(fresh, 0) - fresh
    place = torch.arange(s["positions"].numel(), device="cuda") - first_row[s["token_seq"].long()]
    q = torch.zeros(n, new, h, d, device="cuda")
    q[s["token_seq"].long(), place] = s["qkv"][:, :h * d].float().reshape(-1, h, d)
    q = q.reshape(n, new, kvh, h // kvh, d).permute(0, 2, 3, 1, 4).reshape(n, kvh, h // kvh * new, d)
    sc = torch.matmul(q, k.transpose(2, 3)).reshape(n, kvh, h // kvh, new, longest) * s["scale"]
    if s["softcap"]:
        sc = s["softcap"] * torch.tanh(sc / s["softcap"])
    pos = (lens - fresh)[:, None] + torch.arange(new, device="cuda")[None, :]
    key = torch.arange(longest, device="cuda")
    seen = key[None, None, :] <= pos[:, :, None]
    if s["window"]:
        seen &= pos[:, :, None] - key[None, None, :] < s["window"]
    sc.masked_fill_(~seen[:, None, None], -math.inf)
    sc = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(sc.reshape(n, kvh, -1, longest), v).reshape(n, kvh, h // kvh, new, d) / sc.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, new, h * d)
    return o[s["token_seq"].long(), place].to(dt)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _byte_values():
    """What the 256 bytes of e4m3 stand for."""
    out = []
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = (1.0 + m / 8.0) * 2.0 ** (e - 7) if e else m / 8.0 * 2.0 ** -6
        out.append(math.nan if b & 127 == 127 else -x if b >> 7 else x)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _held(s, which, request, upto):
    """[positions, kv heads, dim] of one request, in 64 bits."""
    page = s["case"]["page"]
    ids = s["table"][int(s["slots"][request])][:-(-upto // page)].long()
    q, e = s[which + "_pages"].view(torch.uint8)[ids], s[which + "_exp"][ids]
    x = _byte_values()[q.long()] * ((e.long() + (1023 - 127)) << 52).view(torch.float64)[..., None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:upto]


def exact(case, seed):
    s = prepare(case, seed)
    kvh, h, d, page = case["kv_heads"], case["heads"], case["dim"], case["page"]
    def two(e):
        return ((e.long() + 1023) << 52).view(torch.float64)

    if case["op"] == "write":
        def stored(x):                                                  # nearest multiple of the step at |x| / 2^e
            a = x.abs().amax(-1, keepdim=True)
            e = torch.frexp(a / LONGEST).exponent                       # a / 448 in [2^(e - 1), 2^e)
            e = torch.where(a == LONGEST * two(e - 1), e - 1, e)
            e = torch.where(a > 0, e, torch.full_like(e, SHORTEST)).clamp_min(SHORTEST)
            y = x / two(e)
            step = two(torch.frexp(y.abs().clamp_min(2.0 ** -6)).exponent - 4)
            return torch.round(y / step) * step * two(e)                # (ties to even)
        x = s["qkv"].double()
        return {"k": stored(x[:, h * d:(h + kvh) * d].reshape(-1, kvh, d)), "v": stored(x[:, (h + kvh) * d:].reshape(-1, kvh, d))}
    if case["op"] == "read":
        out = {}
        for which in ("k", "v"):
            whole = []
            for b, (length, _) in enumerate(s["lens"]):
                x = _held(s, which, b, length)
                pad = torch.zeros(-length % page, kvh, d, dtype=torch.float64, device="cuda")
                whole.append(torch.cat([x, pad]).reshape(-1, page, kvh, d).transpose(1, 2))
            out[which] = torch.cat(whole)
        return out
    out, at = torch.zeros(s["positions"].numel(), h, d, dtype=torch.float64, device="cuda"), 0
    for b, (length, fresh) in enumerate(s["lens"]):
        k, v = _held(s, "k", b, length), _held(s, "v", b, length)
        q = s["qkv"][at:at + fresh, :h * d].double().reshape(fresh, h, d)
        p = torch.arange(length - fresh, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = (j > p) | ((p - j >= s["window"]) if s["window"] else torch.zeros_like(j > p))
        for head in range(h):
            g = head // (h // kvh)
            z = q[:, head] @ k[:, g].T * s["scale"]
            if s["softcap"]:
                z = s["softcap"] * torch.tanh(z / s["softcap"])
            z = z.masked_fill(hidden, -math.inf)
            out[at:at + fresh, head] = torch.softmax(z, dim=-1) @ v[:, g]
        at += fresh
    return out.reshape(-1, h * d)
